"""The paged-cache operators as measured work: rotary positions (`rope`), the
append of new rows to a paged K/V cache (`append_paged`) and the attention of
new tokens over it (`attend_paged`).

`listed()` gives the cases, `draw(rng)` more of the same ranges, `prepare`
what a program has in hand before the call, `run` one call (the plain form,
or the package's where `own` is true), `exact` the same answer in 64 bits and
`work` the bytes and operations that a call cannot do without.
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "flash-attention-cuda_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flashattn_cuda
    return flashattn_cuda


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def rope_case(name, batch, length, heads, kv_heads, dim, rotary, dtype,
              interleaved, inverse, first, factor):
    """`first`: largest position a sequence begins at; `factor`: positions are
    divided by it (linear scaling for a longer context)."""
    return dict(name=name, op="rope", batch=batch, length=length, heads=heads,
                kv_heads=kv_heads, dim=dim, rotary=rotary, dtype=dtype,
                interleaved=interleaved, inverse=inverse, first=first,
                factor=factor)


def append_case(name, batch, new, ragged, past, heads, kv_heads, dim, rotary,
                dtype, interleaved, page, token_major, shape):
    """`new`, `past`: most new tokens and most cached rows of a sequence;
    `ragged`: sequences bring between one and `new` tokens, else all bring
    `new`; `token_major`: pages are (rows, heads, dim), else (heads, rows,
    dim); `shape` seeds the lengths."""
    return dict(name=name, op="append", batch=batch, new=new, ragged=ragged,
                past=past, heads=heads, kv_heads=kv_heads, dim=dim,
                rotary=rotary, dtype=dtype, interleaved=interleaved, page=page,
                token_major=token_major, shape=shape)


def attend_case(name, batch, new, ragged, past, heads, kv_heads, dim, dtype,
                causal, page, token_major, shape):
    return dict(name=name, op="attend", batch=batch, new=new, ragged=ragged,
                past=past, heads=heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype, causal=causal, page=page, token_major=token_major,
                shape=shape)


def listed():
    return [
        # one generation step of a few sequences, nothing else in the call:
        # launch latency
        rope_case("rope_step", 16, 1, 14, 2, 64, 64, "fp16", False, False, 4000, 1.0),
        # a training batch at the 14/2-head, 64-wide shape of the grouped
        # benchmarks, whole head rotated
        rope_case("rope_train", 4, 4096, 14, 2, 64, 64, "bf16", False, False, 0, 1.0),
        # its gradient for a wider model: odd length, neighbouring pairs, half
        # of the head rotated, positions scaled for a long context
        rope_case("rope_gradient", 2, 5001, 32, 8, 128, 64, "fp16", True, True, 120000, 4.0),
        # one token of one sequence: the smallest append
        append_case("append_one", 1, 1, False, 700, 14, 2, 64, 64, "fp16", False, 16, False, 1),
        # a generation step of a full server batch
        append_case("append_batch", 64, 1, False, 1500, 32, 8, 128, 128, "bf16", False, 64, False, 2),
        # prompt chunks of several requests, token-major pages
        append_case("append_chunks", 6, 2500, True, 3000, 32, 8, 128, 128, "bf16", True, 16, True, 3),
        # one token of one short sequence: the smallest attention, latency
        attend_case("attend_one", 1, 1, False, 700, 14, 2, 64, "fp16", True, 16, False, 4),
        # a generation step of a full server batch with ragged contexts
        attend_case("attend_batch", 64, 1, False, 8192, 32, 8, 128, "bf16", True, 64, False, 5),
        # one token of one very long sequence (131072 rows)
        attend_case("attend_long", 1, 1, False, -131071, 14, 2, 64, "fp16", True, 64, False, 6),
        # a few drafted tokens a sequence checked at once, one K/V head per
        # query head
        attend_case("attend_draft", 16, 5, False, 6000, 16, 16, 64, "fp16", True, 32, True, 7),
        # prompts being read beside sequences in generation; a page size that
        # does not divide the key tiles
        attend_case("attend_mixed", 12, 700, True, 3500, 12, 12, 64, "fp16", True, 24, False, 8),
        # one chunk of a long prompt: tensor-bound
        attend_case("attend_chunk", 1, 2048, False, -14336, 32, 8, 128, "bf16", True, 64, False, 9),
    ]


HEADS = [(14, 2), (12, 12), (32, 8), (16, 16), (24, 3), (8, 1), (28, 4),
         (32, 32), (40, 2), (9, 3)]
PAGES = [8, 16, 24, 32, 48, 64, 128, 256]


def spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(
        rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    heads, kv_heads = rng.choice(HEADS)
    dim = rng.choice([64, 128])
    dtype = rng.choice(["fp16", "bf16"])
    rotary = rng.choice([dim, dim, dim // 2, dim // 4])
    page = rng.choice(PAGES)
    shape = rng.randrange(1 << 20)
    if op == "rope":
        batch = spread(rng, 1, 16)
        most = max(1, min(8192, 400000 // (batch * (heads + kv_heads) * dim // 64)))
        c = rope_case("", batch, spread(rng, 1, most), heads, kv_heads, dim,
                      rotary, dtype, rng.random() < 0.5, rng.random() < 0.4,
                      rng.choice([0, 4000, 120000]), rng.choice([1.0, 4.0]))
    elif op == "append":
        batch = spread(rng, 1, 64)
        most = max(1, min(4096, 400000 // (batch * (heads + kv_heads) * dim // 64)))
        c = append_case("", batch, spread(rng, 1, most), rng.random() < 0.6,
                        spread(rng, 1, max(1, 100000 // batch // kv_heads)),
                        heads, kv_heads, dim, rotary, dtype,
                        rng.random() < 0.5, page, rng.random() < 0.5, shape)
    else:
        # half of the draws are generation steps, half bring longer chunks;
        # at most 2^30 scores, and 2^29 cache elements, a call
        batch = spread(rng, 1, 64)
        new = rng.choice([1, spread(rng, 1, 8), spread(rng, 1, 2048),
                          spread(rng, 1, 2048)])
        rows = (1 << 29) // (batch * kv_heads * dim)
        past = spread(rng, 1, max(1, min(65536, rows - 2048)))
        while batch * new * heads * (past + new) > 1 << 30:
            if batch > 1:
                batch = (batch + 1) // 2
            else:
                past = max(1, past // 2)
                new = max(1, new - new // 4)
        c = attend_case("", batch, new, rng.random() < 0.5, past, heads,
                        kv_heads, dim, dtype, rng.random() < 0.85, page,
                        rng.random() < 0.5, shape)
    del c["name"]
    return c


def lengths(case):
    """New tokens and cached rows of each sequence. A negative `past` is the
    rows of every sequence; otherwise they are between none and `past`, and
    the largest is there."""
    rng = random.Random(case["shape"])
    b = case["batch"]
    news = [rng.randint(1, case["new"]) if case["ragged"] else case["new"]
            for _ in range(b)]
    if case["past"] < 0:
        return news, [-case["past"]] * b
    pasts = [rng.randint(0, case["past"]) for _ in range(b)]
    pasts[b // 2] = case["past"]
    return news, pasts


def frequencies(case, device):
    """Radians a position turns each rotated pair by."""
    i = torch.arange(0, case["rotary"], 2, dtype=torch.float64, device=device)
    return 10000.0 ** (-i / case["rotary"]) / case.get("factor", 1.0)


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 2654435761 % (1 << 62) + 17)
    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]

    def normal(*size):
        return torch.randn(*size, generator=gen, device=dev, dtype=dtype)

    if case["op"] == "rope":
        b, n = case["batch"], case["length"]
        first = torch.randint(0, case["first"] + 1, (b, 1), generator=gen,
                              device=dev, dtype=torch.int32)
        positions = (first + torch.arange(n, device=dev, dtype=torch.int32)).contiguous()
        if case["inverse"]:  # gradients, laid out as the attention reads them
            q, k = normal(b, heads, n, dim), normal(b, kv_heads, n, dim)
        else:  # views of one projection's output
            qkv = normal(b, n, heads + 2 * kv_heads, dim).transpose(1, 2)
            q, k = qkv[:, :heads], qkv[:, heads:heads + kv_heads]
        return dict(case=case, q=q, k=k, positions=positions,
                    freqs=frequencies(case, dev))

    news, pasts = lengths(case)
    b, page = case["batch"], case["page"]
    lens = [x + y for x, y in zip(news, pasts)]
    used = [-(-x // page) for x in lens]
    total, width = sum(used), max(used)
    tokens = sum(news)
    qkv = normal(tokens, heads + 2 * kv_heads, dim)
    pool = total + 3
    if case["token_major"]:
        kp = normal(pool, page, kv_heads, dim).transpose(1, 2)
        vp = normal(pool, page, kv_heads, dim).transpose(1, 2)
    else:
        kp, vp = normal(pool, kv_heads, page, dim), normal(pool, kv_heads, page, dim)
    order = torch.randperm(pool, generator=gen, device=dev)[:total].to(torch.int32)
    # the table: each sequence's pages, and -1 where it has none
    column = torch.arange(width, device=dev)
    count = torch.tensor(used, device=dev)
    begin = torch.cumsum(count, 0) - count
    at = (begin[:, None] + column).clamp(max=total - 1)
    table = torch.where(column < count[:, None], order[at],
                        torch.full_like(order[at], -1)).contiguous()
    starts = torch.tensor([0] + news, device=dev).cumsum(0).to(torch.int32)
    seq_lens = torch.tensor(lens, device=dev, dtype=torch.int32)
    s = dict(case=case, k_pages=kp, v_pages=vp, table=table, starts=starts,
             lens=seq_lens, most_new=max(news), most_rows=max(lens))
    if case["op"] == "append":
        s.update(q=qkv[:, :heads], k=qkv[:, heads:heads + kv_heads],
                 v=qkv[:, heads + kv_heads:], freqs=frequencies(case, dev))
    else:
        # rows of a page that nothing was stored in hold anything at all
        last = table.gather(1, (count - 1)[:, None])[:, 0].long()
        free = torch.zeros(pool, page, dtype=torch.bool, device=dev)
        free[last] = torch.arange(page, device=dev) > ((seq_lens - 1) % page)[:, None]
        for pages in (kp, vp):
            pages.masked_fill_(free[:, None, :, None], float("nan"))
        # a few scores of each row stand out
        s.update(q=qkv[:, :heads] * 1.5, scale=dim ** -0.5)
    return s


# ---------------------------------------------------------------------------
# One call
# ---------------------------------------------------------------------------
def run(s):
    return (run_own if own else run_plain)(s, s["case"])


def run_own(s, c):
    fa = package()
    if c["op"] == "rope":
        return fa.rope(s["q"], s["k"], s["positions"], s["freqs"],
                       interleaved=c["interleaved"], inverse=c["inverse"])
    if c["op"] == "append":
        q = fa.append_paged(s["k"], s["v"], s["starts"], s["k_pages"],
                            s["v_pages"], s["table"], s["lens"], q=s["q"],
                            freqs=s["freqs"], interleaved=c["interleaved"])
        return q, s["k_pages"], s["v_pages"]
    return fa.attend_paged(s["q"], s["starts"], s["k_pages"], s["v_pages"],
                           s["table"], s["lens"], s["scale"],
                           causal=c["causal"])


def run_plain(s, c):
    if c["op"] == "rope":
        cos, sin = turn(s["positions"], s["freqs"], c["inverse"])
        return tuple(rotated(x, cos[:, None], sin[:, None], c["interleaved"])
                     for x in (s["q"], s["k"]))
    seq, index = places(s, s["q"].shape[0])
    if c["op"] == "append":
        row = (s["lens"] - s["starts"].diff())[seq] + index
        cos, sin = turn(row, s["freqs"], False)
        q, k = (rotated(x, cos[:, None], sin[:, None], c["interleaved"])
                for x in (s["q"], s["k"]))
        page = s["table"][seq, row // c["page"]].long()
        s["k_pages"][page, :, row % c["page"]] = k
        s["v_pages"][page, :, row % c["page"]] = s["v"]
        return q, s["k_pages"], s["v_pages"]
    return attended(s, c, seq, index)


def places(s, tokens):
    """The sequence of each token, and which of its new tokens it is."""
    t = torch.arange(tokens, device=s["starts"].device)
    seq = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    return seq, t - s["starts"][seq]


def turn(positions, freqs, inverse):
    angle = positions.float()[..., None] * freqs.float()
    return angle.cos(), -angle.sin() if inverse else angle.sin()


def rotated(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    y = x.float()
    if interleaved:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., r:]), -1).to(x.dtype)


def attended(s, c, seq, index):
    b, page, kv, dim = c["batch"], c["page"], c["kv_heads"], c["dim"]
    group, new, rows = c["heads"] // kv, s["most_new"], s["table"].shape[1] * page
    dev = s["q"].device
    key = torch.arange(rows, device=dev)
    there = key < s["lens"][:, None]
    table = s["table"].clamp(min=0).long()

    def whole(pages):  # (batch, kv heads, rows, dim), zero where there is no row
        x = pages[table].transpose(1, 2).reshape(b, kv, rows, dim).float()
        return x.masked_fill_(~there[:, None, :, None], 0.0)

    token = torch.arange(new, device=dev)
    at = (s["starts"][:-1, None] + token).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].float().reshape(b, new, kv, group, dim).permute(0, 2, 3, 1, 4)
    x = q.reshape(b, kv, group * new, dim) @ whole(s["k_pages"]).transpose(-1, -2)
    x = x.mul_(s["scale"]).reshape(b, kv, group, new, rows)
    sees = there[:, None].expand(b, new, rows)
    if c["causal"]:
        place = (s["lens"] - s["starts"].diff())[:, None] + token
        sees = sees & (key <= place[..., None])
    x.masked_fill_(~sees[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top > float("-inf"), top, torch.zeros_like(top))).exp_()
    total = x.sum(-1, keepdim=True)
    o = x.reshape(b, kv, group * new, rows) @ whole(s["v_pages"])
    o = o.reshape(b, kv, group, new, dim) / total.clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(b, new, kv * group, dim)[seq, index].to(s["q"].dtype)


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return tuple(exact_rope(x, s["positions"][:, None], s, case) for x in (s["q"], s["k"]))
    starts, lens, table = (s[x].tolist() for x in ("starts", "lens", "table"))
    page, kv = case["page"], case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if case["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
    for b in range(case["batch"]):
        lo, hi = starts[b], starts[b + 1]
        place = torch.arange(lens[b] - (hi - lo), lens[b], device="cuda")
        pages = torch.tensor(table[b], device="cuda")
        if case["op"] == "append":
            out[lo:hi] = exact_rope(s["q"][lo:hi], place[:, None], s, case)
            k = exact_rope(s["k"][lo:hi], place[:, None], s, case)
            for h in range(kv):
                kp[pages[place // page], h, place % page] = k[:, h]
                vp[pages[place // page], h, place % page] = s["v"][lo:hi, h].double()
            continue
        group = case["heads"] // kv
        pages = pages[:-(-lens[b] // page)]
        for h in range(kv):
            k = s["k_pages"][pages, h].flatten(0, 1)[:lens[b]].double()
            v = s["v_pages"][pages, h].flatten(0, 1)[:lens[b]].double()
            for g in range(h * group, (h + 1) * group):
                x = s["q"][lo:hi, g].double() @ k.T * s["scale"]
                if case["causal"]:
                    x[torch.arange(lens[b], device="cuda") > place[:, None]] = -math.inf
                out[lo:hi, g] = torch.softmax(x, -1) @ v
    return (out, kp, vp) if case["op"] == "append" else out


def exact_rope(x, positions, s, case):
    """Each pair as a complex number, turned by e^(i angle)."""
    r = case["rotary"]
    angle = positions.double()[..., None] * s["freqs"]
    if case.get("inverse"):
        angle = -angle
    y = x.double().clone()
    pair = y[..., :r]
    pair = pair.unflatten(-1, (r // 2, 2)) if case["interleaved"] else \
        pair.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) *
                           torch.polar(torch.ones_like(angle), angle))
    y[..., :r] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
    return y


# ---------------------------------------------------------------------------
# What a call cannot do without
# ---------------------------------------------------------------------------
def work(case):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        tokens = case["batch"] * case["length"]
        return dict(bytes=tokens * ((h + kv) * d * 4 + 4) + case["rotary"] * 4,
                    flops=tokens * (h + kv) * case["rotary"] * 3)
    news, pasts = lengths(case)
    tokens, page = sum(news), case["page"]
    meta = 4 * (2 * case["batch"] + 1) + 4 * sum(-(-(n + p) // page) for n, p in zip(news, pasts))
    if case["op"] == "append":  # q and v once in and out, k too
        return dict(bytes=tokens * (h + 2 * kv) * d * 4 + case["rotary"] * 4 + meta,
                    flops=tokens * (h + kv) * case["rotary"] * 3)
    pairs = sum(n * p + (n * (n + 1) // 2 if case["causal"] else n * n)
                for n, p in zip(news, pasts))
    rows = sum(n + p for n, p in zip(news, pasts))
    return dict(bytes=tokens * h * d * 4 + rows * kv * d * 4 + meta,
                flops=4 * pairs * h * d)
