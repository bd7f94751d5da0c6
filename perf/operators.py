"""Operators of serving several continuations of a prompt, as cases to measure.

The set: an 8-bit key/value cache in pages (one scale for each page, layer and
KV head), written and read back token by token or in chunks; attention over
it; the page operators that let sequences share, fork, extend and free their
pages and that compact the pool; and the log probabilities by which
continuations are scored.

`run` computes each of them in plain torch operations in 32 bits (`own` false)
or through the public entry points of this repository's library (`own` true).
"""
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}  # GGML type ids
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
TINY = 2.0 ** -126


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # One token of one sequence in the middle of a chat: 32 query heads on
        # 4 KV heads of 64 elements (the TinyLlama decode step's attention).
        dict(name="attend one token", op="attend", B=1, rows=1, H=32, KV=4, hd=64, P=64, lo=513, hi=513, window=0,
             type="f32"),
        # A served batch: 64 sequences of different lengths around 1024, one
        # new token each, 32/4 heads of 128 (the 30B-A3B decode step).
        dict(name="attend batch of 64", op="attend", B=64, rows=1, H=32, KV=4, hd=128, P=64, lo=640, hi=1152, window=0,
             type="f32"),
        # Long documents: 4 sequences past 100,000 tokens, 16-bit activations.
        dict(name="attend long contexts", op="attend", B=4, rows=1, H=32, KV=4, hd=128, P=128, lo=100001, hi=131072,
             window=0, type="bf16"),
        # Chunks of prompts of up to 64 tokens (the framework's prefill step)
        # after contexts of some thousand, 14/2 heads of 64, small pages, a
        # sliding window that ends inside a page.
        dict(name="attend prompt chunks", op="attend", B=6, rows=64, H=14, KV=2, hd=64, P=32, lo=1000, hi=4097,
             window=2500, type="f16"),
        # One decode step's keys and values of 64 sequences; the last pages are
        # read back.
        dict(name="append one token each", op="append", B=64, rows=1, KV=4, hd=128, P=64, lo=640, hi=1152, back=64,
             type="f32"),
        # Prompts written into the cache, 16-bit activations, ends inside
        # pages; all of it is read back.
        dict(name="append prompts", op="append", B=8, rows=2048, KV=4, hd=128, P=64, lo=1500, hi=2300, back=2048,
             type="bf16"),
        # A prompt of 513 tokens forked into 16 continuations, each then
        # extended by a token: the shared last page is copied for all but one.
        dict(name="pages fork 16", op="fork", S=16, L=22, KV=4, hd=64, P=64, lo=513, hi=513, parents=1, N=160),
        # Beam search over 8 prompts with 4 beams each: the beams are picked
        # anew and extended.
        dict(name="pages beams", op="fork", S=32, L=48, KV=4, hd=128, P=32, lo=300, hi=700, parents=12, N=900),
        # Half of 64 sequences end; their pages are freed and the pool is
        # compacted.
        dict(name="pages compact", op="compact", S=64, L=48, KV=4, hd=128, P=64, lo=640, hi=1152, N=1100),
        # The score of one decoded token and its 5 alternatives.
        dict(name="logprobs one token", op="logprobs", rows=1, V=32000, k=5, temp=1.0, type="f32", pad=0),
        # A batch's step over a large vocabulary, 20 alternatives each.
        dict(name="logprobs batch of 64", op="logprobs", rows=64, V=151936, k=20, temp=1.0, type="f32", pad=0),
        # A whole prompt scored, 16-bit logits with an odd row length.
        dict(name="logprobs of a prompt", op="logprobs", rows=2047, V=151936, k=4, temp=0.7, type="bf16", pad=3),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One more case of the listed ranges: sizes spread over their logarithm."""
    op = rng.choice(["attend", "attend", "append", "fork", "compact", "logprobs"])
    t = rng.choice(["f32", "f16", "bf16"])
    if op == "logprobs":
        rows, V = _log_int(rng, 1, 2000), _log_int(rng, 500, 151936)
        return dict(op=op, rows=rows, V=V, k=rng.choice([0, 1, 2, 5, 8, 20, 32]), temp=rng.choice([1.0, 0.7, 1.3]),
                    type=t, pad=rng.choice([0, 0, 1, 3, 8]))
    hd = rng.choice([64, 64, 80, 96, 112, 128, 128])
    P = rng.choice([32, 64, 128])
    if op in ("fork", "compact"):
        S, L, KV = _log_int(rng, 2, 64), _log_int(rng, 1, 48), rng.choice([1, 2, 4, 8])
        hi = _log_int(rng, 40, 1200)
        page = 2 * L * KV * P * hd
        while S * (hi // P + 2) * page > 3_300_000_000:
            S, hi = max(2, S * 2 // 3), max(40, hi * 2 // 3)
        lo = max(1, hi * rng.randint(3, 10) // 10)
        N = int(S * (hi // P + 2) * (1.05 + 0.4 * rng.random())) + 3
        c = dict(op=op, S=S, L=L, KV=KV, hd=hd, P=P, lo=lo, hi=hi, N=N)
        if op == "fork":
            c["parents"] = rng.randint(1, S)
        return c
    KV = rng.choice([1, 2, 4, 8, 16])
    if op == "append":
        B, rows = _log_int(rng, 1, 64), _log_int(rng, 1, 2048)
        while B * rows * KV * hd > 8 * 2048 * 4 * 128:
            B, rows = max(1, B // 2), max(1, rows * 3 // 4)
        hi = rows + _log_int(rng, 1, 1500)
        return dict(op=op, B=B, rows=rows, KV=KV, hd=hd, P=P, lo=max(1, hi * rng.randint(3, 10) // 10), hi=hi,
                    back=rows + rng.randint(0, P), type=t)
    group = rng.choice([1, 2, 4, 7, 8, 12])
    B, rows, hi = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 1, 2, 4, 5, 8, 33, 64]), _log_int(rng, 64, 131072)
    while B * hi * KV * hd > 4 * 115000 * 4 * 128 or B * rows * KV * group * hi > 6 * 64 * 14 * 4097:
        B, hi = max(1, B * 2 // 3), max(rows, hi * 3 // 4)
        if B == 1 and hi <= 4097:
            rows = max(1, rows // 2)
            group = max(1, group // 2)
    return dict(op=op, B=B, rows=rows, H=KV * group, KV=KV, hd=hd, P=P, lo=max(1, hi * rng.randint(3, 10) // 10), hi=hi,
                window=rng.choice([0, 0, 0, max(1, hi // 3)]), type=t)


# ----------------------------------------------------------------- inputs --

def _lens(case, n):
    """Lengths of n sequences, spread over lo..hi: the case's, for every seed."""
    lo, hi = case["lo"], case["hi"]
    return [hi if n == 1 else lo + (i * 7919 + 13 * n) % (hi - lo + 1) for i in range(n)]


def _row_counts(case):
    """New tokens of each sequence: `rows` for the first, fewer for some others
    (one at least, and never more than the sequence has)."""
    lens = _lens(case, case["B"])
    return [min(ln, case["rows"] if b % 3 == 0 else max(1, case["rows"] - (b * 5) % case["rows"]))
            for b, ln in enumerate(lens)]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2654435761 % (1 << 62))
    return g


def _codes(g, shape):
    """8-bit codes as a cache holds them: normal values whose largest in a page
    meets 127."""
    n = int(np.prod(shape, dtype=np.int64))
    out = torch.empty(n, dtype=torch.int8, device="cuda")
    step = 1 << 27
    for i in range(0, n, step):
        m = min(step, n - i)
        out[i:i + m] = (torch.randn(m, generator=g, device="cuda") * 30).round_().clamp_(-127, 127).to(torch.int8)
    return out.view(shape)


def _bytes(g, shape):
    """8-bit codes that are only moved: any byte."""
    n = int(np.prod(shape, dtype=np.int64))
    return torch.randint(-2 ** 62, 2 ** 62, ((n + 7) // 8,), generator=g, device="cuda").view(torch.int8)[:n].view(shape)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(g, case, lens, layers, n_pages, max_pages, codes):
    """A pool and page tables in which the sequences' pages lie anywhere."""
    KV, P, hd = case["KV"], case["P"], case["hd"]
    s = {"k": codes(g, (n_pages, layers, KV, P, hd)), "v": codes(g, (n_pages, layers, KV, P, hd)),
         "ks": torch.rand(n_pages, layers, KV, generator=g, device="cuda") * 0.02 + 0.02,
         "vs": torch.rand(n_pages, layers, KV, generator=g, device="cuda") * 0.02 + 0.02}
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    need = [-(-ln // P) for ln in lens]
    table = torch.full((len(lens), max_pages), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    refs[perm[:at].long()] = 1
    s.update(table=table, refs=refs, lens=_i32(lens))
    return s


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "logprobs":
        rows, V, ld = case["rows"], case["V"], case["V"] + case["pad"]
        x = torch.empty(rows, ld, dtype=DTYPES[case["type"]], device="cuda")
        for i in range(0, rows, 256):
            x[i:i + 256] = torch.randn(min(256, rows - i), ld, generator=g, device="cuda") * 2.5
        # Some tokens are barred, as samplers bar them.
        x[:, torch.randint(0, V, (3,), generator=g, device="cuda")] = float("-inf")
        tok = torch.randint(0, V, (rows,), generator=g, device="cuda").to(torch.int32)
        s = {"x": x, "tok": tok, "logprob": torch.empty(rows, device="cuda"),
             "entropy": torch.empty(rows, device="cuda"), "lse": torch.empty(rows, device="cuda"),
             "ids": torch.empty(rows, case["k"], dtype=torch.int32, device="cuda"),
             "top": torch.empty(rows, case["k"], device="cuda")}
    elif op in ("attend", "append"):
        B, KV, P, hd, dt = case["B"], case["KV"], case["P"], case["hd"], DTYPES[case["type"]]
        lens, n = _lens(case, B), _row_counts(case)
        max_pages = -(-max(lens) // P) + 1
        n_pages = sum(-(-ln // P) for ln in lens) + 2
        s = _cache(g, case, lens, 1, n_pages, max_pages, _codes)
        s["start"] = _i32(np.concatenate([[0], np.cumsum(n)]).tolist())
        s["max_len"], s["max_rows"], total = max(lens), max(n), sum(n)
        if op == "attend":
            H = case["H"]
            s["q"] = torch.randn(total, H, hd, generator=g, device="cuda").to(dt)
            s["out"] = torch.empty(total, H, hd, dtype=dt, device="cuda")
            s["lse"] = torch.empty(total, H, device="cuda")
        else:
            # Values of outlying size appear, so that pages' scales grow.
            for name in ("kn", "vn"):
                x = torch.randn(total, KV, hd, generator=g, device="cuda")
                s[name] = (x * (1 + 1.5 * torch.rand(total, KV, 1, generator=g, device="cuda"))).to(dt)
            back = [min(ln, max(m, case["back"])) for ln, m in zip(lens, n)]
            s["back"] = _i32(np.concatenate([[0], np.cumsum(back)]).tolist())
            s["back_rows"], s["back_total"] = max(back), sum(back)
            s["kb"], s["vb"] = (torch.empty(sum(back), KV, hd, device="cuda") for _ in range(2))
    else:
        S, P = case["S"], case["P"]
        max_pages = case["hi"] // P + 2
        if op == "fork":
            # The first `parents` slots hold sequences; every slot takes one of
            # them, in no order, and one token more.
            lens = _lens(case, case["parents"]) + [0] * (S - case["parents"])
            pick = torch.randint(0, case["parents"], (S,), generator=g, device="cuda").to(torch.int32)
        else:
            lens = _lens(case, S)
            pick = torch.arange(S, device="cuda", dtype=torch.int32)
            pick[torch.randperm(S, generator=g, device="cuda")[:S // 2]] = -1
        s = _cache(g, case, lens, case["L"], case["N"], max_pages, _bytes)
        s["pick"] = pick
        for name in ("table", "refs", "lens"):
            s[name + "2"] = torch.empty_like(s[name])
        s["grown"] = torch.empty(S, dtype=torch.int32, device="cuda")
        s["map"] = torch.empty(case["N"], dtype=torch.int32, device="cuda")
        s["live"] = torch.empty(1, dtype=torch.int32, device="cuda")
    s["case"] = case
    if own:
        _handles(s)
    return s


def _package():
    at = os.path.join(os.getcwd(), "quantr-in-c_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import quantr
    return quantr


def _handles(s):
    """What a program of this library keeps beside its tensors: the descriptors
    of its pool, page tables and batch, and a workspace."""
    q, case = _package(), s["case"]
    s["lib"] = q
    if case["op"] == "logprobs":
        n = q.logprobs_workspace_bytes(case["rows"], case["V"], case["k"])
    else:
        s["pool"] = q.Kv8Pool.of(s["k"], s["v"], s["ks"], s["vs"])
        s["tables"] = q.Kv8Tables.of(s["table"], s["lens"], s["refs"])
        if case["op"] == "attend":
            s["batch"] = q.Kv8Batch(None, s["start"].data_ptr(), case["B"], s["max_rows"])
            n = q.kv8_attend_workspace_bytes(s["pool"], s["batch"], case["H"], s["max_len"])
        elif case["op"] == "append":
            s["batch"] = q.Kv8Batch(None, s["start"].data_ptr(), case["B"], s["max_rows"])
            s["batch_back"] = q.Kv8Batch(None, s["back"].data_ptr(), case["B"], s["back_rows"])
            n = 0
        else:
            s["tables2"] = q.Kv8Tables.of(s["table2"], s["lens2"], s["refs2"])
            n = q.kv8_pages_workspace_bytes(s["pool"], s["tables"])
    s["ws"] = torch.zeros(max(n, 256), dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------- plain forms --

def _rows_of(start, lens, total):
    """Sequence, and position in it, of each row of a ragged batch whose rows
    are the sequences' last tokens."""
    r = torch.arange(total, device="cuda")
    b = torch.searchsorted(start, r.to(torch.int32), right=True) - 1
    return b, lens[b].long() - (start[b + 1] - start[b]) + (r - start[b])


def _plain_attend(s):
    case = s["case"]
    KV, hd, P, H, W = case["KV"], case["hd"], case["P"], case["H"], case["window"]
    B, R, G, T = case["B"], s["max_rows"], case["H"] // case["KV"], s["table"].shape[1] * case["P"]
    page = s["table"].clamp(min=0).long()
    keys = s["k"][:, 0][page].float() * s["ks"][:, 0][page][..., None, None]
    vals = s["v"][:, 0][page].float() * s["vs"][:, 0][page][..., None, None]
    keys, vals = (x.permute(0, 2, 1, 3, 4).reshape(B, KV, T, hd) for x in (keys, vals))
    total = s["q"].shape[0]
    b, pos = _rows_of(s["start"], s["lens"], total)
    i = torch.arange(total, device="cuda") - s["start"][b]
    q = torch.zeros(B, R, H, hd, device="cuda")
    q[b, i] = s["q"].float()
    q = q.view(B, R, KV, G, hd).permute(0, 2, 1, 3, 4).reshape(B, KV, R * G, hd)
    x = torch.matmul(q, keys.transpose(2, 3)) * (hd ** -0.5)
    # Row i of a sequence sees the positions up to its own, `window` at most.
    own_pos = (s["lens"] - (s["start"][1:] - s["start"][:-1]))[:, None] + torch.arange(R, device="cuda")
    t = torch.arange(T, device="cuda")
    seen = (t <= own_pos[..., None]) & (t < s["lens"][:, None, None])
    if W:
        seen &= t > own_pos[..., None] - W
    seen = seen[:, None, :, None, :]
    x = x.view(B, KV, R, G, T).masked_fill(~seen, float("-inf"))
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
    total_p = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, KV, R * G, T), vals).view(B, KV, R, G, hd)
    o = torch.where(total_p > 0, o / total_p, 0.0)
    lse = (m + torch.log(total_p))[..., 0]
    o = o.permute(0, 2, 1, 3, 4).reshape(B, R, H, hd)[b, i].to(s["out"].dtype)
    return {"out": o, "lse": lse.permute(0, 2, 1, 3).reshape(B, R, H)[b, i]}


def _append_plain(codes, scales, new, s, P):
    """Writes the rows of `new` behind their sequences: a page that begins with
    new rows gets the scale of its largest magnitude; the scale of a page that
    had rows is doubled until the new ones fit, its codes being rounded anew."""
    start, lens = s["start"].long(), s["lens"].long()
    n = start[1:] - start[:-1]
    first = lens - n
    M = (s["max_rows"] + P - 2) // P + 1
    at = first[:, None] // P + torch.arange(M, device="cuda")
    valid = at * P < lens[:, None]
    page = s["table"].long().gather(1, at.clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    pos = at[..., None] * P + torch.arange(P, device="cuda")
    is_new = (pos >= first[:, None, None]) & (pos < lens[:, None, None])
    row = (start[:-1, None, None] + pos - first[:, None, None]).clamp(0, new.shape[0] - 1)
    x = torch.where(is_new[..., None, None], new[row].float(), 0.0).permute(0, 1, 3, 2, 4)  # B M KV P hd
    top = x.abs().amax((-1, -2))
    old_s, old = scales[:, 0][page], codes[:, 0][page]
    had = ((at * P < first[:, None]) & valid)[..., None]
    fresh = torch.maximum(top / torch.full_like(top, 127.0), torch.full_like(top, TINY))
    room = old_s * 127.0
    mt, et = torch.frexp(top)
    mr, er = torch.frexp(room)
    j = torch.where(top <= room, 0, et - er + (mt > mr).int()).clamp(min=0)
    scale = torch.where(had, torch.ldexp(old_s, j), fresh)
    coded = (x * (torch.ones_like(scale) / scale)[..., None, None]).round().clamp(-127, 127)
    again = torch.where(had[..., None, None], torch.ldexp(old.float(), -j[..., None, None]).round(), old.float())
    out = torch.where(is_new[:, :, None, :, None], coded, again).to(torch.int8)
    codes[page[valid], 0] = out[valid]
    scales[page[valid], 0] = scale[valid]


def _plain_append(s):
    P = s["case"]["P"]
    _append_plain(s["k"], s["ks"], s["kn"], s, P)
    _append_plain(s["v"], s["vs"], s["vn"], s, P)
    b, pos = _rows_of(s["back"], s["lens"], s["back_total"])
    page = s["table"][b, pos // P].long()
    return {"k": s["k"][page, 0, :, pos % P].float() * s["ks"][page, 0][..., None],
            "v": s["v"][page, 0, :, pos % P].float() * s["vs"][page, 0][..., None]}


def _plain_select(s):
    """Slot i takes the pages of slot pick[i] (none: -1)."""
    pick, P = s["pick"].long(), s["case"]["P"]
    has = pick >= 0
    lens = torch.where(has, s["lens"][pick.clamp(min=0)], 0)
    kept = torch.arange(s["table"].shape[1], device="cuda") < ((lens + P - 1) // P)[:, None]
    table = torch.where(kept, s["table"][pick.clamp(min=0)], -1)
    refs = torch.zeros(s["refs"].numel() + 1, dtype=torch.int32, device="cuda")
    refs.index_add_(0, torch.where(kept, table, refs.numel() - 1).view(-1).long(),
                    torch.ones(table.numel(), dtype=torch.int32, device="cuda"))
    return table, lens, refs[:-1]


def _move(s, dst, src):
    for name in ("k", "v", "ks", "vs"):
        s[name][dst] = s[name][src]


def _words(s):
    """The pool's contents, which page operators move unseen, as 32-bit words."""
    return {name: s[name].view(-1).view(torch.int32) for name in ("k", "v", "ks", "vs")}


def _plain_fork(s):
    P, S = s["case"]["P"], s["case"]["S"]
    table, lens, refs = _plain_select(s)
    # One token more for every sequence, in the order of the slots.
    tail = table.gather(1, ((lens - 1).clamp(min=0) // P)[:, None].long())[:, 0]
    inside = (lens % P != 0)
    before = torch.tril(torch.ones(S, S, dtype=torch.bool, device="cuda"), -1)
    rank = ((tail[:, None] == tail[None, :]) & inside[None, :] & before).sum(1)
    copied = inside & (refs[tail.clamp(min=0).long()] - rank > 1)
    fresh = ~inside
    need = (copied | fresh).long()
    upto = need.cumsum(0)
    free = torch.argsort((refs != 0).int(), stable=True)
    grown = (upto <= (refs == 0).sum()) & (lens // P < table.shape[1])
    got = free[(upto - 1).clamp(0, free.numel() - 1)]
    copied, fresh = copied & grown, fresh & grown
    src = tail.clamp(min=0).long()
    _move(s, torch.where(copied, got, src), src)
    row, col = torch.arange(S, device="cuda"), (lens // P).clamp(max=table.shape[1] - 1).long()
    table[row, col] = torch.where(copied | fresh, got.to(torch.int32), table[row, col])
    one = (copied | fresh).int()
    refs.index_add_(0, got, one)
    refs.index_add_(0, src, -copied.int())
    return {"table": table, "lens": lens + grown.int(), "refs": refs, "grown": grown.int(), **_words(s)}


def _plain_compact(s):
    N = s["case"]["N"]
    table, lens, refs = _plain_select(s)
    used = refs > 0
    live = used.sum()
    index = torch.arange(N, device="cuda")
    src, dst = index[used & (index >= live)], index[~used & (index < live)]
    to = torch.where(used, index, -1)
    to[src] = dst
    _move(s, dst, src)
    refs[dst] = refs[src]
    refs = torch.where(index < live, refs, 0)
    table = torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), -1)
    return {"table": table, "lens": lens, "refs": refs, "map": to.to(torch.int32), "live": live.to(torch.int32).view(1),
            **_words(s)}


def _plain_logprobs(s):
    case = s["case"]
    V, k = case["V"], case["k"]
    raw = s["x"][:, :V].float()
    x = raw * torch.tensor(1.0 / case["temp"], device="cuda")
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    lp = x - lse
    entropy = -(torch.where(e > 0, lp, 0.0) * e).sum(1) / total[:, 0]
    # Alternatives by value, of equal values the lower index first.
    bits = raw.view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + (V - 1 - torch.arange(V, device="cuda"))
    ids = V - 1 - (torch.topk(order, k, dim=1).values & 0xFFFFFFFF)
    return {"logprob": lp.gather(1, s["tok"].long()[:, None])[:, 0], "entropy": entropy, "lse": lse[:, 0],
            "ids": ids.to(torch.int32), "top": lp.gather(1, ids)}


PLAIN = {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact,
         "logprobs": _plain_logprobs}


# --------------------------------------------------------------- own calls --

def _own_attend(s):
    case = s["case"]
    ld = case["H"] * case["hd"]
    s["lib"].kv8_attend_dev(s["out"].data_ptr(), ld, s["q"].data_ptr(), ld, TYPE_IDS[case["type"]], case["H"],
                            s["pool"], s["tables"], s["batch"], 0, case["hd"] ** -0.5, s["max_len"],
                            s["ws"].data_ptr(), s["ws"].numel(), window=case["window"], lse=s["lse"].data_ptr())
    return {"out": s["out"], "lse": s["lse"]}


def _own_append(s):
    case = s["case"]
    ld = case["KV"] * case["hd"]
    s["lib"].kv8_append_dev(s["kn"].data_ptr(), ld, s["vn"].data_ptr(), ld, TYPE_IDS[case["type"]], s["pool"],
                            s["tables"], s["batch"], 0)
    s["lib"].kv8_read_dev(s["kb"].data_ptr(), ld, s["vb"].data_ptr(), ld, TYPE_IDS["f32"], s["pool"], s["tables"],
                          s["batch_back"], 0)
    return {"k": s["kb"], "v": s["vb"]}


def _own_fork(s):
    lib = s["lib"]
    lib.kv8_select_dev(s["tables2"], s["tables"], s["pick"].data_ptr(), s["pool"])
    lib.kv8_extend_dev(s["pool"], s["tables2"], None, None, s["case"]["S"], s["ws"].data_ptr(), s["ws"].numel(),
                       grown=s["grown"].data_ptr())
    return {"table": s["table2"], "lens": s["lens2"], "refs": s["refs2"], "grown": s["grown"], **_words(s)}


def _own_compact(s):
    lib = s["lib"]
    lib.kv8_select_dev(s["tables2"], s["tables"], s["pick"].data_ptr(), s["pool"])
    lib.kv8_compact_dev(s["pool"], s["tables2"], s["map"].data_ptr(), s["live"].data_ptr(), s["ws"].data_ptr(),
                        s["ws"].numel())
    return {"table": s["table2"], "lens": s["lens2"], "refs": s["refs2"], "map": s["map"], "live": s["live"],
            **_words(s)}


def _own_logprobs(s):
    case = s["case"]
    s["lib"].logprobs_dev(s["x"].data_ptr(), s["x"].shape[1], TYPE_IDS[case["type"]], case["rows"], case["V"],
                          s["tok"].data_ptr(), s["logprob"].data_ptr(), s["entropy"].data_ptr(), case["k"],
                          s["ids"].data_ptr(), s["top"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(),
                          temperature=case["temp"], lse=s["lse"].data_ptr())
    return {"logprob": s["logprob"], "entropy": s["entropy"], "lse": s["lse"], "ids": s["ids"], "top": s["top"]}


OWN = {"attend": _own_attend, "append": _own_append, "fork": _own_fork, "compact": _own_compact,
       "logprobs": _own_logprobs}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------- floor --

def work(case):
    """Bytes: each input read once, each output written once (page operators:
    the pages that move, read and written). Flops: products and sums of the
    definition."""
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["V"]
        return {"bytes": n * SIZES[case["type"]] + case["rows"] * (16 + 8 * case["k"]), "flops": 4 * n}
    KV, hd, P = case["KV"], case["hd"], case["P"]
    if op in ("attend", "append"):
        lens, n = _lens(case, case["B"]), _row_counts(case)
        size = SIZES[case["type"]]
        if op == "append":
            rows = sum(n)
            back = sum(min(ln, max(m, case["back"])) for ln, m in zip(lens, n))
            return {"bytes": 2 * KV * hd * (rows * (size + 1) + back * (1 + 4)), "flops": 4 * KV * hd * (rows + back)}
        W = case["window"] or max(lens)
        tokens = sum(min(ln, W + m - 1) for ln, m in zip(lens, n))
        seen = sum(min(ln - m + 1 + i, W) for ln, m in zip(lens, n) for i in range(m))
        return {"bytes": 2 * KV * tokens * (hd + 4 / P) + sum(n) * case["H"] * (2 * hd * size + 4),
                "flops": 4 * case["H"] * hd * seen}
    page = 2 * case["L"] * KV * (P * hd + 4)
    small = 4 * (2 * case["S"] * (case["hi"] // P + 2) + 2 * case["N"])
    if op == "fork":
        lens = [_lens(case, case["parents"])[i % case["parents"]] for i in range(case["S"])]
        moved = max(0, sum(ln % P != 0 for ln in lens) - case["parents"])
    else:
        live = sum(-(-ln // P) for ln in _lens(case, case["S"])) / 2
        moved = live * (1 - live / case["N"])
    return {"bytes": 2 * moved * page + small, "flops": 0}


# -------------------------------------------------------------- definition --

def exact(case, seed):
    """The definitions in 64 bits, one sequence and one page at a time."""
    op = case["op"]
    if op in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    if op == "logprobs":
        got = {"logprob": [], "entropy": [], "lse": [], "top": []}
        for i in range(0, case["rows"], 64):
            x = s["x"][i:i + 64, :case["V"]].double() / case["temp"]
            lse = torch.logsumexp(x, 1)
            lp = x - lse[:, None]
            got["lse"].append(lse)
            got["logprob"].append(lp[torch.arange(x.shape[0]), s["tok"][i:i + 64].long()])
            got["entropy"].append(-torch.nan_to_num(lp.exp() * lp, nan=0.0).sum(1))
            got["top"].append(lp.sort(1, descending=True).values[:, :case["k"]])
        return {"ids": None, **{n: torch.cat(v) for n, v in got.items()}}
    P, lens, start, table = case["P"], s["lens"].tolist(), s["start"].tolist(), s["table"].tolist()
    if op == "attend":
        G, W = case["H"] // case["KV"], case["window"]
        out = torch.empty(start[-1], case["H"], case["hd"], dtype=torch.float64, device="cuda")
        lse = torch.empty(start[-1], case["H"], dtype=torch.float64, device="cuda")
        for b, ln in enumerate(lens):
            pages = table[b][:-(-ln // P)]
            n = start[b + 1] - start[b]
            pos = torch.arange(ln - n, ln, device="cuda")[:, None]
            t = torch.arange(ln, device="cuda")
            hidden = (t > pos) | (t <= pos - W) if W else t > pos
            for h in range(case["KV"]):
                k, v = (s[c][pages, 0, h].double() * s[z][pages, 0, h].double()[:, None, None]
                        for c, z in (("k", "ks"), ("v", "vs")))
                k, v = k.reshape(-1, case["hd"])[:ln], v.reshape(-1, case["hd"])[:ln]
                for g in range(h * G, h * G + G):
                    x = s["q"][start[b]:start[b + 1], g].double() @ k.T / case["hd"] ** 0.5
                    x[hidden] = float("-inf")
                    lse[start[b]:start[b + 1], g] = torch.logsumexp(x, 1)
                    out[start[b]:start[b + 1], g] = torch.softmax(x, 1) @ v
        return {"out": out, "lse": lse}
    back, got = s["back"].tolist(), {}
    for c, z, x, name in (("k", "ks", "kn", "k"), ("v", "vs", "vn", "v")):
        rows = []
        for b, ln in enumerate(lens):
            first, seq = ln - (start[b + 1] - start[b]), []
            for at in range((ln - (back[b + 1] - back[b])) // P, -(-ln // P)):
                lo, hi = max(at * P, first), min(at * P + P, ln)
                page = table[b][at]
                code, scale = s[c][page, 0].double(), s[z][page, 0].double()
                if hi > lo:
                    new = s[x][start[b] + lo - first:start[b] + hi - first].double().permute(1, 0, 2)
                    top = new.abs().amax((1, 2))
                    if lo > at * P:
                        grow = torch.exp2(torch.ceil(torch.log2(top / (scale * 127))).clamp(min=0))
                        scale, code = scale * grow, (code / grow[:, None, None]).round()
                    else:
                        scale = top / 127
                    code[:, lo - at * P:hi - at * P] = (new / scale[:, None, None]).round().clamp(-127, 127)
                seq.append((code * scale[:, None, None]).permute(1, 0, 2))
            began = (ln - (back[b + 1] - back[b])) // P * P
            rows.append(torch.cat(seq)[ln - (back[b + 1] - back[b]) - began:ln - began])
        got[name] = torch.cat(rows)
    return got
