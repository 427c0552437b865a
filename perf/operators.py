"""The operators of one serving step over an 8-bit paged KV cache, in a plain form and as the framework's calls.

A step of a batch of sequences: `plan` gives the new tokens their pages and slots, `append` quantises their K and V
rows into the pages, `attend` runs attention over the pages, `draw` picks the next tokens from the logits.

A page holds 32 positions of one sequence: codes [page][kv head][K, V][32][head_dim] in 8 bits and one f32 scale for
each [page][kv head][K, V]; a position's values are code * scale.
"""
import math
import os
import sys

import torch

own = False

PAGE = 32
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOP = {"e4m3": 448.0, "i8": 127.0}


def listed():
    return [
        # 32 sequences, one new token each, some of them at a page's end: the step of batched decoding
        dict(name="plan decode 32", op="plan", seqs=32, pad=0, new="one", most=2048, short=False),
        # a busy server's step: prefill chunks of many lengths among decoding sequences, rows padded
        dict(name="plan mixed 512", op="plan", seqs=512, pad=333, new="mixed", most=4096, short=False),
        # one new row of each of 32 sequences, the activations in f32 as the engine keeps them (8B shape)
        dict(name="append decode 32", op="append", seqs=32, rows=1, heads=8, dim=128, fmt="e4m3", dtype="f32", pad=0),
        # a prompt of 8192 tokens (7B shape)
        dict(name="append prompt 8192", op="append", seqs=1, rows=8192, heads=4, dim=128, fmt="i8", dtype="bf16", pad=0),
        # prompts of odd lengths for a large batch (70B's 8 KV heads), a padded batch
        dict(name="append ragged 24", op="append", seqs=24, rows=1999, heads=8, dim=128, fmt="e4m3", dtype="f16", pad=77),
        # one sequence, one token, the 0.5B shape: latency
        dict(name="attend decode 1", op="attend", seqs=1, rows=1, most=1024, q_heads=14, heads=2, dim=64, fmt="e4m3",
             dtype="f32", window=0, pad=0),
        # 32 sequences of ragged lengths, the 8B shape
        dict(name="attend decode 32", op="attend", seqs=32, rows=1, most=4096, q_heads=32, heads=8, dim=128, fmt="e4m3",
             dtype="bf16", window=0, pad=0),
        # few long sequences, the 7B shape
        dict(name="attend long 4", op="attend", seqs=4, rows=1, most=131072, q_heads=28, heads=4, dim=128, fmt="i8",
             dtype="bf16", window=0, pad=0),
        # several rows a sequence (drafted tokens to verify) inside a sliding window, the 70B shape
        dict(name="attend verify 8", op="attend", seqs=8, rows=5, most=8192, q_heads=64, heads=8, dim=128, fmt="i8",
             dtype="f16", window=4096, pad=3),
        # a prompt's chunks over what was read before, the 7B shape
        dict(name="attend chunk 2", op="attend", seqs=2, rows=1024, most=8192, q_heads=28, heads=4, dim=128, fmt="e4m3",
             dtype="bf16", window=0, pad=0),
        # one sequence's next token: the engine's f32 logits of the 7B vocabulary, top-k and top-p
        dict(name="draw 1", op="draw", rows=1, vocab=152064, dtype="f32", mode="topk", mask=False),
        # a batch of requests that each bring their own settings, the 8B vocabulary
        dict(name="draw 64", op="draw", rows=64, vocab=128256, dtype="bf16", mode="mixed", mask=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "draw"])
    fmt, dtype = rng.choice(["e4m3", "i8"]), rng.choice(["f32", "f16", "bf16"])
    if op == "plan":
        new = rng.choice(["one", "mixed"])
        return dict(op=op, seqs=_log(rng, 1, 4096 if new == "one" else 512), pad=rng.choice([0, 1, _log(rng, 1, 500)]), new=new,
                    most=_log(rng, 40, 4096), short=rng.random() < 0.25)
    if op == "append":
        heads, dim = rng.choice([1, 2, 4, 8, 16]), rng.choice([16, 64, 64, 80, 96, 128, 128])
        rows = _log(rng, 1, 8192)
        seqs = _log(rng, 1, max(1, min(256, 16384 // rows * 128 * 8 // (dim * heads) // 2 or 1)))
        return dict(op=op, seqs=seqs, rows=rows, heads=heads, dim=dim, fmt=fmt, dtype=dtype, pad=rng.choice([0, 0, 5, 64]))
    if op == "attend":
        heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 4, 4, 7, 7, 8, 8, 12])
        dim = rng.choice([16, 64, 64, 80, 96, 128, 128, 128])
        rows = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 1024)])
        most = _log(rng, max(rows, 33), 65536 if rows < 4 else 8192)
        # what the plain form holds at once: keys and values in f32, and the scores
        room = min(2**28 // (most * heads * dim), 2**28 // (most * rows * heads * group))
        seqs = _log(rng, 1, max(1, min(128, room)))
        if rows > 16:
            seqs = min(seqs, max(1, 2**32 // (rows * most * heads * group)))
        return dict(op=op, seqs=seqs, rows=rows, most=most, q_heads=heads * group, heads=heads, dim=dim, fmt=fmt, dtype=dtype,
                    window=rng.choice([0, 0, 0, _log(rng, 1, most)]), pad=rng.choice([0, 0, 1, 9]))
    vocab = _log(rng, 100, 160000)
    return dict(op=op, rows=_log(rng, 1, min(256, 8200000 // vocab)), vocab=vocab, dtype=dtype,
                mode=rng.choice(["topk", "topp", "minp", "plain", "greedy", "mixed", "mixed"]), mask=rng.random() < 0.3)


# ---------------------------------------------------------------- inputs ----
def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _spread(n, lo, hi):
    """n lengths over [lo, hi], hi among them: the same ones whatever the seed, so that totals stay."""
    return [hi - int((hi - lo + 1) * (i * 0.6180339887498949 % 1.0)) for i in range(n)]


def _lengths(g, n, lo, hi):
    """_spread in an order of the seed's."""
    return torch.tensor(_spread(n, lo, hi), dtype=torch.int32, device="cuda")[torch.randperm(n, generator=g, device="cuda")]


def _chunks(case):
    """New tokens of each sequence in a `plan` case: one, or a quarter of them a chunk and a few nothing."""
    n = case["seqs"]
    if case["new"] == "one":
        return [1] * n
    return [x if i % 4 == 0 else int(i % 20 != 1) for i, x in enumerate(_spread(n, 1, 511))]


def _codes(g, shape, fmt):
    """Codes of K and V values: normally distributed, the page's largest near the type's largest."""
    out = torch.empty(shape, dtype=torch.uint8, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        x = torch.empty(n, device="cuda").normal_(generator=g)
        if fmt == "e4m3":
            flat[i:i + n] = x.mul_(110.0).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            flat[i:i + n] = x.mul_(30.0).clamp_(-127, 127).round_().to(torch.int8).view(torch.uint8)
    return out


def _scales(g, shape, fmt):
    """Powers of two about 1 / (a code's standard deviation), spread as heads' and pages' magnitudes are."""
    e = torch.randint(-8, -5, shape, generator=g, device="cuda") if fmt == "e4m3" else \
        torch.randint(-6, -3, shape, generator=g, device="cuda")
    return torch.pow(2.0, e.float())


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op = case["op"]
    if op == "plan":
        n, most = case["seqs"], case["most"]
        lens = _lengths(g, n, 0, most)
        add = torch.tensor(_chunks(case), dtype=torch.int32, device="cuda")[torch.randperm(n, generator=g, device="cuda")]
        old, new = (lens + 31) // 32, (lens + add + 31) // 32
        ld = (most + 512 + 31) // 32
        pages = int(new.sum()) + 64
        perm = torch.randperm(pages, generator=g, device="cuda").int()
        table = torch.full((n, ld), -1, dtype=torch.int32, device="cuda")
        held = torch.arange(ld, device="cuda")[None, :] < old[:, None]
        n_old = int(old.sum())
        table[held] = perm[:n_old]
        need = int((new - old).sum())
        free = perm[n_old:].contiguous()
        if case["short"]:  # the pool runs out part-way
            free = free[:max(1, need // 2)].contiguous()
        rows = sum(_chunks(case)) + case["pad"]
        s.update(lens=lens, add=add, table=table, free=free, n_free=torch.tensor([free.numel()], dtype=torch.int32, device="cuda"),
                 n_rows=rows)
        i32 = dict(dtype=torch.int32, device="cuda")
        s.update(lens_out=torch.zeros(n, **i32), first=torch.zeros(n + 1, **i32), pos=torch.zeros(rows, **i32),
                 seq=torch.zeros(rows, **i32), slots=torch.zeros(rows, dtype=torch.int64, device="cuda"),
                 status=torch.zeros(2, **i32))
    elif op == "append":
        n, H, D, fmt = case["seqs"], case["heads"], case["dim"], case["fmt"]
        add = _lengths(g, n, max(1, case["rows"] // 2), case["rows"])
        off = torch.randint(0, 32, (n,), generator=g, device="cuda", dtype=torch.int32)  # rows already in the last page
        touched = (off + add + 31) // 32
        n_pages = sum((31 + a + 31) // 32 for a in _spread(n, max(1, case["rows"] // 2), case["rows"])) + 1
        perm = torch.randperm(n_pages, generator=g, device="cuda")
        T = int(add.sum())
        first = torch.cumsum(add, 0) - add
        seq = torch.repeat_interleave(torch.arange(n, device="cuda"), add.long())
        p = torch.arange(T, device="cuda") - first[seq] + off[seq]
        slots = perm[(torch.cumsum(touched, 0) - touched)[seq] + p // 32] * 32 + p % 32
        T += case["pad"]
        slots = torch.cat([slots, torch.full((case["pad"],), -1, dtype=torch.int64, device="cuda")])
        # activations: normal, with a few large channels (K) and rows of different magnitude
        mag = torch.exp2(torch.randint(-2, 3, (T, 1, 1), generator=g, device="cuda").float())
        big = 1 + 7 * (torch.rand((1, H, D), generator=g, device="cuda") < 0.03).float()
        s["k"] = (torch.empty((T, H, D), device="cuda").normal_(generator=g) * mag * big).to(DT[case["dtype"]])
        s["v"] = (torch.empty((T, H, D), device="cuda").normal_(generator=g) * mag).to(DT[case["dtype"]])
        s["slots"] = slots
        s["codes"] = _codes(g, (n_pages, H, 2, PAGE, D), fmt)
        s["scales"] = _scales(g, (n_pages, H, 2), fmt)
        s["n_pages"] = n_pages
    elif op == "attend":
        n, H, D, fmt = case["seqs"], case["heads"], case["dim"], case["fmt"]
        add = _lengths(g, n, max(1, case["rows"] // 2), case["rows"])
        lens = _lengths(g, n, max(case["rows"], case["most"] // 2), case["most"])
        pages = (lens + 31) // 32
        ld = int(pages.max())
        total = int(pages.sum())
        n_pages = total + 7
        perm = torch.randperm(n_pages, generator=g, device="cuda").int()
        table = torch.full((n, ld), -1, dtype=torch.int32, device="cuda")
        table[torch.arange(ld, device="cuda")[None, :] < pages[:, None]] = perm[:total]
        first = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        first[1:] = torch.cumsum(add, 0)
        T = int(first[-1]) + case["pad"]
        s["codes"] = _codes(g, (n_pages, H, 2, PAGE, D), fmt)
        s["scales"] = _scales(g, (n_pages, H, 2), fmt)
        s["q"] = (1.5 * torch.empty((T, case["q_heads"], D), device="cuda").normal_(generator=g)).to(DT[case["dtype"]])
        s["out"] = torch.zeros_like(s["q"])
        s.update(lens=lens, first=first, table=table, n_pages=n_pages, n_rows=T, max_rows=case["rows"])
    else:
        n, V = case["rows"], case["vocab"]
        # logits: a broad bulk, a few likely tokens above it
        x = torch.empty((n, V), device="cuda").normal_(generator=g).mul_(2.0)
        top = torch.randint(0, V, (n, 24), generator=g, device="cuda")
        x.scatter_add_(1, top, torch.rand((n, 24), generator=g, device="cuda") * 12)
        s["logits"] = x.to(DT[case["dtype"]])
        t = 0.6 + 0.7 * torch.rand(n, generator=g, device="cuda")
        k = torch.zeros(n, dtype=torch.int32, device="cuda")
        p = torch.ones(n, device="cuda")
        m = torch.zeros(n, device="cuda")
        mode = case["mode"]
        which = torch.randint(0, 5, (n,), generator=g, device="cuda") if mode == "mixed" else \
            torch.full((n,), ["topk", "topp", "minp", "plain", "greedy"].index(mode), device="cuda")
        k = torch.where(which == 0, torch.randint(1, 200, (n,), generator=g, device="cuda", dtype=torch.int32), k)
        p = torch.where(which <= 1, 0.8 + 0.18 * torch.rand(n, generator=g, device="cuda"), p)
        m = torch.where(which == 2, 0.01 + 0.1 * torch.rand(n, generator=g, device="cuda"), m)
        t = torch.where(which == 4, torch.zeros_like(t), t)
        # {temperature, top_k, top_p, min_p}, 16 bytes a row
        s["params"] = torch.stack([t, k.view(torch.float32), p, m], 1).contiguous()
        s["u"] = torch.rand(n, generator=g, device="cuda")
        s["mask"] = (torch.rand((n, V), generator=g, device="cuda") < 0.8).to(torch.uint8) if case["mask"] else None
        s["tokens"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        s["logprob"] = torch.zeros(n, device="cuda")
    if own:
        sm = _smotor()
        if op in ("append", "attend"):
            s["cache"] = sm.Kv8Cache(s["codes"].data_ptr(), s["scales"].data_ptr(), s["n_pages"], case["heads"], case["dim"],
                                     sm.KV8_E4M3 if case["fmt"] == "e4m3" else sm.KV8_I8)
        if op == "attend":
            s["ws"] = sm.Kv8Workspace()
    return s


def _smotor():
    path = os.path.join(os.getcwd(), "siliceo-motor_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import smotor
    return smotor


# ------------------------------------------------------------ plain forms ----
def _plan_plain(s):
    lens, add, table, free = s["lens"].long(), s["add"].long(), s["table"], s["free"]
    n, ld = table.shape
    T = s["n_rows"]
    n_free = s["n_free"].long()
    good = (lens >= 0) & (add >= 0)
    rows = torch.where(good, add, 0)
    end = torch.cumsum(rows, 0)
    start = end - rows
    good &= (lens + add <= ld * PAGE) & (end <= T)
    old = (lens.clamp(min=0) + 31) // PAGE
    need = torch.where(good, (lens + add + 31) // PAGE - old, 0)
    upto = torch.cumsum(need, 0)
    good &= (need == 0) | (upto <= n_free)
    given = torch.where(good, need, 0)
    before = upto - need
    col = torch.arange(ld, device=table.device)[None, :]
    fresh = good[:, None] & (col >= old[:, None]) & (col < (old + given)[:, None])
    at = (n_free - 1 - (before[:, None] + col - old[:, None])).clamp(0, max(0, free.numel() - 1))
    table.copy_(torch.where(fresh, free[at], table))
    t = torch.arange(T, device=table.device)
    seq = torch.searchsorted(end, t, right=True)
    inside = seq < n
    q = seq.clamp(max=n - 1)
    valid = inside & good[q]
    pos = lens[q] + t - start[q]
    page = table[q, (pos // PAGE).clamp(0, ld - 1)].long()
    slots = torch.where(valid, page * PAGE + pos % PAGE, -1)
    s["slots"].copy_(slots)
    s["pos"].copy_(torch.where(valid, pos, -1))
    s["seq"].copy_(torch.where(inside, seq, -1))
    s["first"][:1] = 0
    s["first"][1:] = end
    s["lens_out"].copy_(torch.where(good, lens + add, -1))
    s["status"][0:1] = n_free - given.sum()
    s["status"][1:2] = n - good.sum()


def _values(codes, scales, fmt):
    x = codes.view(torch.float8_e4m3fn).float() if fmt == "e4m3" else codes.view(torch.int8).float()
    return x * scales[..., None, None]


def _append_plain(s):
    """A page's scale becomes the smallest power of two that holds its rows' largest value, if that is more than it was."""
    fmt, slots, codes, scales = s["fmt"], s["slots"], s["codes"], s["scales"]
    P, H, _, _, D = codes.shape
    x = torch.stack([s["k"], s["v"]], 2).float()  # [T, H, 2, D]
    page = torch.where(slots >= 0, slots // PAGE, P)  # rows without a slot go to a page behind the last
    top = torch.zeros((P + 1, H, 2), device=x.device)
    top.scatter_reduce_(0, page[:, None, None].expand(-1, H, 2), x.abs().amax(-1), "amax")
    low = torch.full((P + 1,), PAGE, dtype=torch.int64, device=x.device)
    low.scatter_reduce_(0, page, slots % PAGE, "amin")  # the page's first new row: those before it stay
    m, e = torch.frexp(top[:P] / TOP[fmt])  # top / M = m * 2^e, m in [0.5, 1)
    need = torch.exp2(torch.where(m > 0.5, e, e - 1).clamp(min=-100).float())
    need = torch.where(top[:P] > 0, need, 2.0**-100)
    low = low[:P]
    kept = torch.where((low == 0)[:, None, None], need, torch.maximum(scales, need))
    new = torch.where((low < PAGE)[:, None, None], kept, scales)
    old = _values(codes, scales / new, fmt)  # every row in units of its page's new scale
    # rows at and behind the page's first new row: written below, or as they were
    stay = torch.arange(PAGE, device=x.device)[None, :] >= low[:, None]
    typed = codes.view(torch.float8_e4m3fn) if fmt == "e4m3" else codes.view(torch.int8)
    enc = _encode(old, fmt)
    enc = torch.where(stay[:, None, None, :, None], typed.view(torch.uint8), enc)
    spare = torch.cat([new, torch.ones_like(new[:1])])
    rows = _encode(x / spare[page][..., None], fmt)  # [T, H, 2, D]
    full = torch.cat([enc, enc.new_zeros((1, H, 2, PAGE, D))])
    full[page, :, :, slots % PAGE] = rows
    codes.copy_(full[:P])
    scales.copy_(new)


def _encode(x, fmt):
    if fmt == "e4m3":
        return x.to(torch.float8_e4m3fn).view(torch.uint8)
    return x.round().to(torch.int8).view(torch.uint8)


def _attend_plain(s):
    n, R = s["lens"].numel(), s["max_rows"]
    H, D, G = s["heads"], s["dim"], s["q_heads"] // s["heads"]
    lens, first = s["lens"].long(), s["first"].long()
    add = first[1:] - first[:-1]
    page = s["table"].long().clamp(min=0)
    kv = _values(s["codes"][page], s["scales"][page], s["fmt"])  # [n, pages, H, 2, 32, D]
    kv = kv.permute(3, 0, 2, 1, 4, 5).reshape(2, n, H, -1, D)
    L = kv.shape[3]
    i = torch.arange(R, device=page.device)
    live = i[None, :] < add[:, None]
    row = (first[:-1, None] + i[None, :]).clamp(max=s["n_rows"] - 1)
    q = s["q"][row].float()  # [n, R, Hq, D]
    q = q.view(n, R, H, G, D).permute(0, 2, 3, 1, 4).reshape(n, H, G * R, D)
    a = torch.matmul(q, kv[0].transpose(-1, -2)).view(n, H, G, R, L).mul_(1 / math.sqrt(D))
    at = (lens - add)[:, None] + i[None, :]
    j = torch.arange(L, device=page.device)
    see = (j[None, None, :] <= at[:, :, None]) & (j[None, None, :] < lens[:, None, None])
    if s["window"]:
        see &= j[None, None, :] > at[:, :, None] - s["window"]
    a.masked_fill_(~see[:, None, None], -math.inf)
    a.sub_(a.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    z = a.sum(-1, keepdim=True)
    o = torch.matmul(a.view(n, H, G * R, L), kv[1]).view(n, H, G, R, D)
    o = torch.where(z > 0, o / z, 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, R, H * G, D).to(s["q"].dtype)
    s["out"][row[live]] = o[live]


def _draw_plain(s):
    x = s["logits"].float()
    n, V = x.shape
    t, p, m = s["params"][:, 0].double(), s["params"][:, 2].double(), s["params"][:, 3].double()
    k = s["params"].view(torch.int32)[:, 1].long()
    if s["mask"] is not None:
        x = x.masked_fill(s["mask"] == 0, -math.inf)
    x, at = torch.sort(x, dim=1, descending=True, stable=True)
    d = x.double() - x[:, :1].double()
    w = torch.exp(d / torch.where(t > 0, t, 1.0)[:, None])
    rank = torch.arange(V, device=x.device)[None, :]
    k = torch.where(t > 0, torch.where(k > 0, k, V), 1)
    w = torch.where(rank < k[:, None], w, 0.0)
    below = torch.cumsum(w, 1) - w
    keep = (rank == 0) | ((below < p[:, None] * w.sum(1, keepdim=True)) | (p[:, None] >= 1)) & (w >= m[:, None])
    w = torch.zeros_like(w).scatter_(1, at, torch.where(keep, w, 0.0))  # back in the vocabulary's order
    c = torch.cumsum(w, 1)
    total = c[:, -1:]
    token = (c <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    s["tokens"].copy_(token[:, 0])
    s["logprob"].copy_(torch.log(w.gather(1, token) / total)[:, 0])


def run(state):
    s = state
    op = s["op"]
    if own:
        sm = _smotor()
        stream = torch.cuda.current_stream().cuda_stream
        if op == "plan":
            sm.kv_plan(s["seqs"], s["lens"].data_ptr(), s["add"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1],
                       s["free"].data_ptr(), s["n_free"].data_ptr(), s["n_rows"], s["lens_out"].data_ptr(), s["first"].data_ptr(),
                       s["slots"].data_ptr(), s["status"].data_ptr(), pos=s["pos"].data_ptr(), seq=s["seq"].data_ptr(), stream=stream)
        elif op == "append":
            s["cache"].append(s["k"].data_ptr(), s["v"].data_ptr(), _type(sm, s), s["slots"].numel(), s["slots"].data_ptr(),
                              stream=stream)
        elif op == "attend":
            s["cache"].attend(s["ws"], s["q"].data_ptr(), s["out"].data_ptr(), _type(sm, s), s["n_rows"], s["q_heads"], s["seqs"],
                              s["lens"].data_ptr(), s["first"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1],
                              window=s["window"], stream=stream)
        else:
            sm.draw(s["logits"].data_ptr(), _type(sm, s), s["rows"], s["vocab"], s["params"].data_ptr(), s["u"].data_ptr(),
                    s["tokens"].data_ptr(), logprobs=s["logprob"].data_ptr(),
                    mask=0 if s["mask"] is None else s["mask"].data_ptr(), stream=stream)
    else:
        {"plan": _plan_plain, "append": _append_plain, "attend": _attend_plain, "draw": _draw_plain}[op](s)
    return _outputs(s)


def _type(sm, s):
    return {"f32": sm.F32, "f16": sm.F16, "bf16": sm.BF16}[s["dtype"]]


def _outputs(s):
    op = s["op"]
    if op == "plan":
        return {k: s[k] for k in ("table", "lens_out", "first", "slots", "pos", "seq", "status")}
    if op == "append":  # a position's values: code * scale
        return {"codes": s["codes"].view(torch.float8_e4m3fn if s["fmt"] == "e4m3" else torch.int8), "scales": s["scales"]}
    if op == "attend":
        return {"out": s["out"]}
    return {"tokens": s["tokens"], "logprob": s["logprob"]}


# ------------------------------------------------------------------- work ----
def work(case):
    op = case["op"]
    if op == "plan":
        n = case["seqs"]
        rows = sum(_chunks(case)) + case["pad"]
        return {"bytes": 16 * n + 16 * rows + 8 * (rows // PAGE), "flops": 0}
    if op == "append":
        rows = sum(_spread(case["seqs"], max(1, case["rows"] // 2), case["rows"]))
        size = torch.empty(0, dtype=DT[case["dtype"]]).element_size()
        return {"bytes": 2 * rows * case["heads"] * case["dim"] * (size + 1) + 8 * rows, "flops": 0}
    if op == "attend":
        n = case["seqs"]
        rows = sum(_spread(n, max(1, case["rows"] // 2), case["rows"]))
        length = sum(_spread(n, max(case["rows"], case["most"] // 2), case["most"])) / n
        per = rows / n
        if case["window"]:
            length = min(length, case["window"] + per - 1)
        seen = max(1.0, min(length - (per - 1) / 2, case["window"] or length))
        size = torch.empty(0, dtype=DT[case["dtype"]]).element_size()
        return {"bytes": 2 * int(n * length) * case["heads"] * case["dim"] + 2 * rows * case["q_heads"] * case["dim"] * size,
                "flops": 4.0 * rows * seen * case["q_heads"] * case["dim"]}
    size = torch.empty(0, dtype=DT[case["dtype"]]).element_size()
    return {"bytes": case["rows"] * case["vocab"] * (size + int(case["mask"])), "flops": 0}


# ------------------------------------------------------------------ exact ----
def exact(case, seed):
    """What run() returns, from the definitions in 64 bits, one sequence (or row) after another."""
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    return {"plan": lambda _: None, "append": _append_exact, "attend": _attend_exact, "draw": _draw_exact}[case["op"]](s)


def _append_exact(s):
    codes = s["codes"].view(torch.float8_e4m3fn if s["fmt"] == "e4m3" else torch.int8).double()
    scales = s["scales"].double()
    k, v, slots = s["k"].double(), s["v"].double(), s["slots"].tolist()
    if len(slots) > 60000:
        return None
    i = 0
    while i < len(slots):
        if slots[i] < 0:
            i += 1
            continue
        j = i + 1
        while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] % PAGE:
            j += 1
        page, a = divmod(slots[i], PAGE)
        b = a + j - i
        for which, x in ((0, k), (1, v)):
            r = x[i:j].transpose(0, 1)  # [H, rows, D]
            top = r.abs().amax((1, 2))
            need = torch.where(top > 0, torch.ceil(torch.log2(top / TOP[s["fmt"]])), -100.0).clamp(min=-100)
            need = torch.exp2(need)
            new = torch.maximum(scales[page, :, which], need) if a else need
            near = (codes[page, :, which, :a] * (scales[page, :, which] / new)[:, None, None], r / new[:, None, None])
            for (c, d), y in zip(((0, a), (a, b)), near):
                codes[page, :, which, c:d] = y.float().to(torch.float8_e4m3fn).double() if s["fmt"] == "e4m3" else y.round()
            scales[page, :, which] = new
        i = j
    if s["fmt"] == "i8":
        codes = codes.to(torch.int8)
    return {"codes": codes, "scales": scales}


def _attend_exact(s):
    H, D, G = s["heads"], s["dim"], s["q_heads"] // s["heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens, first = s["lens"].tolist(), s["first"].tolist()
    for i, L in enumerate(lens):
        a, b = first[i], first[i + 1]
        if a == b:
            continue
        page = s["table"][i, :(L + 31) // 32].long()
        pos = torch.arange(L - (b - a), L, device="cuda")
        j = torch.arange(L, device="cuda")
        see = j[None, :] <= pos[:, None]
        if s["window"]:
            see &= j[None, :] > pos[:, None] - s["window"]
        for h in range(H):
            c, f = s["codes"][page, h], s["scales"][page, h].double()
            c = (c.view(torch.float8_e4m3fn) if s["fmt"] == "e4m3" else c.view(torch.int8)).double() * f[:, :, None, None]
            kk, vv = (c[:, w].reshape(-1, D)[:L] for w in (0, 1))
            for r0 in range(0, b - a, 256):
                r1 = min(b - a, r0 + 256)
                q = s["q"][a + r0:a + r1, h * G:(h + 1) * G].double()
                x = torch.einsum("rgd,ld->rgl", q, kk) / math.sqrt(D)
                x = torch.softmax(x.masked_fill(~see[r0:r1, None, :], -math.inf), -1)
                out[a + r0:a + r1, h * G:(h + 1) * G] = torch.einsum("rgl,ld->rgd", x, vv)
    return {"out": out}


def _draw_exact(s):
    n = s["rows"]
    tokens, logp = [], []
    par, ks = s["params"].tolist(), s["params"].view(torch.int32)[:, 1].tolist()
    u = s["u"].tolist()
    for i in range(n):
        t, _, p, m = par[i]
        x = s["logits"][i].double()
        ids = torch.arange(x.numel(), device=x.device)
        if s["mask"] is not None:
            ids = ids[s["mask"][i] != 0]
            x = x[ids]
        order = torch.sort(x, descending=True, stable=True).indices
        if t <= 0:
            tokens.append(int(ids[order[0]]))
            logp.append(0.0)
            continue
        if ks[i] > 0:
            order = order[:ks[i]]
        w = torch.exp((x[order] - x[order[0]]) / t)
        c = torch.cumsum(w, 0)
        cut = w.numel() if p >= 1 else max(1, int(((c - w) < p * c[-1]).sum()))
        cut = min(cut, max(1, int((w >= m).sum())))
        kept = torch.sort(order[:cut]).values
        y = torch.exp((x[kept] - x[order[0]]) / t)
        c = torch.cumsum(y, 0)
        at = min(int((c <= u[i] * c[-1]).sum()), cut - 1)
        tokens.append(int(ids[kept[at]]))
        logp.append(float(torch.log(y[at] / c[-1])))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprob": torch.tensor(logp, dtype=torch.float64)}
