"""Cases and plain forms of the operators around a paged key / value cache.

K and V rows of many sequences lie in pages of ``ps`` rows, [pages, Hkv, ps, D]; row p of sequence b is row
p % ps of page ``table[b, p // ps]``. Four operators work on it:

* ``append``  the K and V rows of new tokens, one per sequence or whole prompts packed back to back, go into
              the pages, K rotated by its position on the way, and the tokens' queries are rotated;
* ``prompt``  causal attention of whole prompts packed back to back, before or without a cache;
* ``chunk``   the same of the last tokens of every sequence over all of its rows in the pages;
* ``decode``  one token of every sequence over its rows; groups of sequences share their first rows' pages.

With positions p (0-based) the rotation of a row x is x * cos[p] + turned(x) * sin[p], where turned(x) is
(-x[D/2:], x[:D/2]); attention is softmax over j <= p of q.k_j / sqrt(D), applied to v_j; query head h reads
K / V head h // (Hq / Hkv).

``run`` computes an operator in elementary torch operations (``own`` false) or through
``deltaattention_b200.ops`` (``own`` true), ``exact`` in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one sequence's token: latency alone
        dict(name="append 1 fp16 d64", op="append", B=1, lo=1, hi=1, past=700, Hq=8, H=8, D=64, ps=16, dtype="fp16",
             tables="fp16", layout="head"),
        # a token of each of 64 sequences
        dict(name="append 64 bf16", op="append", B=64, lo=1, hi=1, past=4000, Hq=32, H=8, D=128, ps=16, dtype="bf16",
             tables="fp32", layout="head"),
        # a batch of prompts of different lengths
        dict(name="append 16 prompts bf16", op="append", B=16, lo=999, hi=6001, past=0, Hq=32, H=8, D=128, ps=64,
             dtype="bf16", tables="fp32", layout="row"),
        # one short prompt
        dict(name="prompt 500 fp16 d64", op="prompt", B=1, lo=500, hi=500, Hq=8, H=8, D=64, dtype="fp16"),
        # a batch of short and ordinary prompts
        dict(name="prompt 12 ragged bf16", op="prompt", B=12, lo=99, hi=4000, Hq=32, H=8, D=128, dtype="bf16"),
        # one prompt of 32k tokens
        dict(name="prompt 32k bf16", op="prompt", B=1, lo=32768, hi=32768, Hq=32, H=8, D=128, dtype="bf16"),
        # the next turn of one conversation
        dict(name="chunk 300 over 2k fp16 d64", op="chunk", B=1, lo=300, hi=300, past=2000, Hq=16, H=4, D=64, ps=32,
             dtype="fp16", layout="row"),
        # pieces of four long prompts, beside what the earlier pieces left in the cache
        dict(name="chunk 4x512 over 16k bf16", op="chunk", B=4, lo=512, hi=512, past=16000, Hq=32, H=8, D=128, ps=16,
             dtype="bf16", layout="head"),
        # a token of one short sequence
        dict(name="decode 1x2k fp16 d64", op="decode", B=1, groups=0, prefix=0, lo=1900, hi=1900, Hq=16, H=4, D=64, ps=16,
             dtype="fp16", layout="head"),
        # a token of each of 48 sequences of very different lengths, nothing shared
        dict(name="decode 48 ragged bf16", op="decode", B=48, groups=0, prefix=0, lo=500, hi=12001, Hq=32, H=8, D=128,
             ps=16, dtype="bf16", layout="head"),
        # 64 answers over one document of 32k tokens
        dict(name="decode 64 share 32k bf16", op="decode", B=64, groups=1, prefix=32000, lo=1, hi=1000, Hq=32, H=8, D=128,
             ps=16, dtype="bf16", layout="head"),
        # four documents with a few sequences each, seven query heads per K / V head
        dict(name="decode 4x24 share 8k bf16", op="decode", B=96, groups=4, prefix=8000, lo=100, hi=2000, Hq=28, H=4,
             D=128, ps=64, dtype="bf16", layout="row"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "prompt", "chunk", "decode", "decode"])
    D = rng.choice([64, 128])
    H = rng.choice([1, 2, 4, 8, 8])
    Hq = H * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    dtype = rng.choice(["bf16", "fp16"])
    paged = dict(ps=rng.choice([16, 32, 64, 128]), layout=rng.choice(["head", "row"]))
    base = dict(op=op, Hq=Hq, H=H, D=D, dtype=dtype)
    if op == "append":
        if rng.random() < 0.4:
            return dict(base, B=_log(rng, 1, 256), lo=1, hi=1, past=rng.randint(0, 8000), tables=rng.choice(["fp32", dtype]),
                        **paged)
        hi = _log(rng, 1, 16000)
        return dict(base, B=max(1, min(_log(rng, 1, 32), 50000 // hi)), lo=rng.choice([hi, hi // 3]), hi=hi,
                    past=rng.choice([0, 0, 77, 2000]), tables=rng.choice(["fp32", dtype]), **paged)
    if op == "prompt":
        hi = _log(rng, 1, 32000)
        most = int(2 ** 30 * 32 * 128 / (hi * hi * Hq * D))
        return dict(base, B=max(1, min(_log(rng, 1, 24), most)), lo=rng.choice([hi, hi // 8]), hi=hi)
    if op == "chunk":
        hi, past = _log(rng, 1, 4000), _log(rng, 1, 32000)
        most = int(2 ** 30 * 32 * 128 / (2 * hi * (hi + past) * Hq * D))
        return dict(base, B=max(1, min(_log(rng, 1, 16), most, 300000 // past)), lo=rng.choice([hi, hi // 8]), hi=hi, past=past,
                    **paged)
    groups = rng.choice([0, 1, 1, 2, 5])
    hi = _log(rng, 1, 4000 if groups else 32000)
    pages = 0 if not groups else _log(rng, 1, 48000 // paged["ps"])
    prefix = pages * paged["ps"]
    B = max(groups, 1, min(_log(rng, 1, 200), 2000000 * 1024 // ((hi + prefix) * H * D)))
    return dict(base, B=B, groups=groups, prefix=prefix, lo=rng.choice([hi, hi // 8, 0]), hi=hi, **paged)


# ------------------------------------------------------------------------------------ inputs
def _lengths(case, seed=0):
    """Every sequence's new (append, prompt, chunk) or own (decode) tokens, as the program that packs them knows
    them: the case's lengths, lo and hi among them, in an order that goes by the seed."""
    lo, hi, rng = case["lo"], case["hi"], random.Random(case["B"])
    n = [lo, hi] + [rng.randint(lo, hi) for _ in range(case["B"] - 2)] if case["B"] > 1 else [hi]
    random.Random(int(seed)).shuffle(n)
    return n


def _starts(n):
    return torch.tensor([0] + n, device="cuda").cumsum(0).to(torch.int32)


def _rows(g, T, H, D, dtype, key):
    """K rows, with an offset per head and channel, or V rows, as a layer's projections give them."""
    x = torch.randn((T, H, D), generator=g, device="cuda")
    if key:
        return x.add_(torch.randn((1, H, D), generator=g, device="cuda")).to(dtype)
    return x.mul_(0.5).to(dtype)


def _pages(g, case, pages, dtype):
    """K and V pages that hold rows everywhere, as in a cache that has been in use for a while."""
    H, ps, D = case["H"], case["ps"], case["D"]
    k = _rows(g, pages * ps, H, D, dtype, True).view(pages, ps, H, D)
    v = _rows(g, pages * ps, H, D, dtype, False).view(pages, ps, H, D)
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    return (k, v) if case["layout"] == "row" else (k.contiguous(), v.contiguous())


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, B, Hq, H, D, dtype = case["op"], case["B"], case["Hq"], case["H"], case["D"], DTYPES[case["dtype"]]
    n = _lengths(case, seed)
    s = dict(op=op, n=n)
    if op == "decode":
        ps, groups = case["ps"], case["groups"]
        of = [b * groups // B for b in range(B)]  # a sequence's group: neighbours, nearly equally many
        first = case["prefix"] // ps if groups else 0
        own_pages = [-(-x // ps) for x in n]
        total = groups * first + sum(own_pages)
        order = torch.randperm(max(total, 1), generator=g, device="cuda").to(torch.int32)
        table = torch.zeros((B, first + max(own_pages + [1])), device="cuda", dtype=torch.int32)
        at = groups * first
        for b in range(B):
            table[b, :first] = order[of[b] * first:(of[b] + 1) * first]
            table[b, first:first + own_pages[b]] = order[at:at + own_pages[b]]
            at += own_pages[b]
        s["k"], s["v"] = _pages(g, case, max(total, 1), dtype)
        s["q"] = (1.5 * torch.randn((B, Hq, D), generator=g, device="cuda")).to(dtype)
        s["lengths"] = torch.tensor([first * ps + x for x in n], device="cuda", dtype=torch.int32)
        s["prefix_cu"] = s["prefix_lengths"] = None
        if groups:
            s["prefix_cu"] = _starts([of.count(i) for i in range(groups)])
            s["prefix_lengths"] = torch.full((groups,), first * ps, device="cuda", dtype=torch.int32)
        return dict(s, table=table)
    T = sum(n)
    s["cu"] = _starts(n)
    if op == "prompt":
        s["q"] = (1.5 * torch.randn((T, Hq, D), generator=g, device="cuda")).to(dtype)
        return dict(s, k=_rows(g, T, H, D, dtype, True), v=_rows(g, T, H, D, dtype, False))
    ps = case["ps"]
    lens = [case["past"] + x for x in n]
    s["lens"], s["lengths"] = lens, torch.tensor(lens, device="cuda", dtype=torch.int32)
    most = -(-max(lens + [1]) // ps)
    s["table"] = torch.randperm(B * most, generator=g, device="cuda").to(torch.int32).view(B, most)
    s["k"], s["v"] = _pages(g, case, B * most, dtype)
    if op == "chunk":
        s["q"] = (1.5 * torch.randn((T, Hq, D), generator=g, device="cuda")).to(dtype)
        return s
    # queries, keys and values side by side, as one projection gives them
    x = torch.randn((T, (Hq + 2 * H) * D), generator=g, device="cuda").to(dtype)
    s["q"], s["k_new"], s["v_new"] = (t.unflatten(1, (-1, D)) for t in x.split([Hq * D, H * D, H * D], 1))
    s["one_each"] = case["lo"] == case["hi"] == 1
    angle = torch.arange(most * ps, device="cuda").double()[:, None] * 5e5 ** (
        -torch.arange(0, D, 2, device="cuda").double() / D)
    angle = torch.cat([angle, angle], 1)
    s["cos"], s["sin"] = angle.cos().to(DTYPES[case["tables"]]), angle.sin().to(DTYPES[case["tables"]])
    return s


# -------------------------------------------------------------------------------- plain forms
def _attend(q, k, v, first):
    """Rows ``first``.. of a sequence, q [n, Hq, D], over its K and V rows [H, L, D], causal; 32 bits."""
    n, Hq, D = q.shape
    H, L, _ = k.shape
    out = torch.empty((n, Hq, D), device=q.device)
    step = max(1, 2 ** 28 // (Hq * L))
    for i in range(0, n, step):
        x = q[i:i + step].float().view(-1, H, Hq // H, D).permute(1, 2, 0, 3)
        m, end = x.shape[2], first + min(n, i + step)
        w = x.reshape(H, -1, D) @ k[:, :end].transpose(1, 2) * D ** -0.5
        w = w.view(H, Hq // H, m, end)
        p = torch.arange(first + i, first + i + m, device=q.device)
        w = w.masked_fill_(torch.arange(end, device=q.device) > p[:, None], -math.inf)
        w = w.sub_(w.amax(-1, keepdim=True)).exp_()
        w = w.div_(w.sum(-1, keepdim=True))
        o = w.view(H, -1, end) @ v[:, :end]
        out[i:i + m] = o.view(H, Hq // H, m, D).permute(2, 0, 1, 3).reshape(m, Hq, D)
    return out


def _plain_prompt(s):
    parts = [_attend(q, k.float().transpose(0, 1).contiguous(), v.float().transpose(0, 1).contiguous(), 0)
             for q, k, v in zip(*(s[x].split(s["n"]) for x in "qkv"))]
    return torch.cat(parts).to(s["q"].dtype)


def _gathered(pages, table):
    """The rows [.., H, rows, D] of the sequences' pages, in 32 bits."""
    return pages[table.long()].transpose(-4, -3).flatten(-3, -2).float()


def _plain_chunk(s):
    parts = [_attend(q, _gathered(s["k"], t)[:, :L], _gathered(s["v"], t)[:, :L], L - len(q))
             for q, t, L in zip(s["q"].split(s["n"]), s["table"], s["lens"])]
    return torch.cat(parts).to(s["q"].dtype)


def _plain_decode(s):
    B, Hq, D = s["q"].shape
    k = _gathered(s["k"], s["table"])
    H, L = k.shape[1:3]
    w = s["q"].float().view(B, H, Hq // H, D) @ k.transpose(2, 3) * D ** -0.5
    del k
    live = (torch.arange(L, device=w.device) < s["lengths"][:, None])[:, None, None]
    w = w.masked_fill_(~live, -math.inf)
    w = torch.where(live, w.sub_(w.amax(-1, keepdim=True)).exp_(), 0.0)
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-30)
    return (w @ _gathered(s["v"], s["table"])).view(B, Hq, D).to(s["q"].dtype)


def _rotated(x, cos, sin):
    h = x.shape[-1] // 2
    x, cos, sin = x.float(), cos.float()[:, None], sin.float()[:, None]
    return x * cos + torch.cat([-x[..., h:], x[..., :h]], -1) * sin


def _plain_append(s):
    cu, T = s["cu"].long(), s["q"].shape[0]
    t = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    p = s["lengths"].long()[b] - (cu[b + 1] - t)
    ps = s["k"].shape[2]
    page, row = s["table"].long()[b, p // ps], p % ps
    cos, sin = s["cos"][p], s["sin"][p]
    s["k"][page, :, row] = _rotated(s["k_new"], cos, sin).to(s["k"].dtype)
    s["v"][page, :, row] = s["v_new"]
    return _rotated(s["q"], cos, sin).to(s["q"].dtype)


# --------------------------------------------------------------------------------- the passes
def run(s):
    if own:
        from deltaattention_b200 import ops
    op = s["op"]
    if op == "append":
        if own:
            q = ops.paged_append(s["k_new"], s["v_new"], ops.PagedKV(s["k"], s["v"]), s["table"], s["lengths"],
                                 cu_seqlens=None if s["one_each"] else s["cu"], cos=s["cos"], sin=s["sin"], q=s["q"])
        else:
            q = _plain_append(s)
        return dict(q=q, k=s["k"], v=s["v"])
    if op == "prompt":
        return ops.flash_varlen(s["q"], s["k"], s["v"], s["cu"]) if own else _plain_prompt(s)
    if op == "chunk":
        if own:
            return ops.flash_paged(s["q"], ops.PagedKV(s["k"], s["v"]), s["table"], s["lengths"], s["cu"])
        return _plain_chunk(s)
    if own:
        return ops.decode_attention_paged(s["q"], ops.PagedKV(s["k"], s["v"]), s["table"], s["lengths"],
                                          prefix_cu=s["prefix_cu"], prefix_lengths=s["prefix_lengths"])
    return _plain_decode(s)


def work(case):
    op, B, Hq, H, D = case["op"], case["B"], case["Hq"], case["H"], case["D"]
    lens, row = _lengths(case), 2 * D
    n = sum(lens) / B
    if op == "append":  # K, V and Q rows in and out, the tables' rows
        width = 4 if case["tables"] == "fp32" else 2
        rows = min(B * n, case["past"] + case["hi"])
        return dict(bytes=B * n * row * 2 * (2 * H + Hq) + rows * 2 * D * width, flops=B * n * D * 3 * (H + Hq))
    if op == "decode":
        shared = case["prefix"] if case["groups"] else 0
        kv = (case["groups"] * shared + B * n) * H * row * 2
        return dict(bytes=kv + 2 * B * Hq * row, flops=4 * D * Hq * B * (shared + n))
    past = case.get("past", 0)
    pairs = sum(x * past + x * (x + 1) // 2 for x in lens)
    return dict(bytes=B * (n * 2 * Hq + (n + past) * 2 * H) * row, flops=4 * D * Hq * pairs)


# -------------------------------------------------------------------------------- in 64 bits
def _exact_heads(q, k, v, see):
    """One K / V head: q [n, G, D], k and v [L, D]; row i sees the first ``see``[i] rows. In 64 bits."""
    n, G, D = q.shape
    k, v = k.double(), v.double()
    out = torch.zeros((n, G, D), dtype=torch.float64, device=q.device)
    if not len(k):
        return out
    step = max(1, 2 ** 27 // (G * len(k)))
    at = torch.arange(len(k), device=q.device)
    for i in range(0, n, step):
        z = torch.einsum("ngd,ld->ngl", q[i:i + step].double(), k) / math.sqrt(D)
        hidden = (at >= see[i:i + step, None])[:, None]
        z = torch.softmax(torch.where(hidden, -math.inf, z), -1)
        out[i:i + step] = torch.einsum("ngl,ld->ngd", torch.where(hidden, 0.0, z), v)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op, Hq, H, D, B = case["op"], case["Hq"], case["H"], case["D"], case["B"]
    G, q = Hq // H, s["q"]
    if op == "append":
        ps = case["ps"]
        out = dict(q=torch.empty(q.shape, dtype=torch.float64, device="cuda"), k=s["k"].double(), v=s["v"].double())
        at = 0
        for b, n in enumerate(s["n"]):
            for x, to in ((s["q"], "q"), (s["k_new"], "k"), (s["v_new"], "v")):
                x = x[at:at + n].double()
                p = torch.arange(s["lens"][b] - n, s["lens"][b], device="cuda")
                if to != "v":
                    a, c = x[..., :D // 2], x[..., D // 2:]
                    cos, sin = s["cos"][p].double()[:, None], s["sin"][p].double()[:, None]
                    x = torch.cat([a * cos[..., :D // 2] - c * sin[..., :D // 2],
                                   c * cos[..., D // 2:] + a * sin[..., D // 2:]], -1)
                if to == "q":
                    out["q"][at:at + n] = x
                else:
                    out[to][s["table"][b].long()[p // ps], :, p % ps] = x
            at += n
        return out
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    at = 0
    for b in range(B):
        n = 1 if op == "decode" else s["n"][b]
        if op == "prompt":
            k, v, L = s["k"][at:at + n], s["v"][at:at + n], n
        else:
            L = int(s["lengths"][b])
            p = torch.arange(L, device="cuda")
            page, row = s["table"][b].long()[p // case["ps"]], p % case["ps"]
            k, v = s["k"][page, :, row], s["v"][page, :, row]
        see = L - n + 1 + torch.arange(n, device="cuda")
        for h in range(H):
            if n and L:
                out[at:at + n, h * G:(h + 1) * G] = _exact_heads(q[at:at + n, h * G:(h + 1) * G], k[:, h], v[:, h], see)
        at += n
    return out
