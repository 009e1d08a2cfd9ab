"""Cases and plain forms of the operators around a decode history held in 4 bits.

A packed decode history (anchors with run-length counts, as the delta selection leaves them) is
kept in 4-bit codes with one scale and one zero per 32 elements, next to the exact window of
recent tokens in 16 bits. Four operators work on it:

* ``handoff``  a prefill's packed K and V rows are put into 4 bits, and read back;
* ``append``   the token that leaves the exact window is merged into the last anchor or appended;
* ``attend``   one token's attention over history and window, with the attention weight that every
               entry drew added to its ``mass``;
* ``evict``    every head is cut to its ``budget`` heaviest entries, in place and in order.

The 4-bit form of a row x of D elements, in groups g of 32:

    zero  = min(x_g) rounded down to bf16
    scale = (max(x_g) - zero) / 15 rounded to bf16
    code  = clamp(round_half_even((x - zero) / scale), 0, 15), 0 where scale = 0
    value = zero + scale * code

A row's codes are D/8 words of 32 bits: word t * (D/32) + g holds, from its lowest bits up, the
codes of elements 32 g + 8 t .. 32 g + 8 t + 7 (t = 0..3). A row's scales are its D/32 scales,
then its D/32 zeros.

``run`` computes an operator in elementary torch operations (``own`` false) or through
``deltaattention_b200.ops`` (``own`` true), ``exact`` in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a 2k-token prompt of 8 heads at one anchor in four: the smallest hand-off of a layer
        dict(name="handoff 2k fp16 d64", op="handoff", B=1, H=8, N=512, D=64, dtype="fp16", layout="head"),
        # one layer of a 32k-token prompt at one anchor in four, rows as the projection lays them out
        dict(name="handoff 32k bf16", op="handoff", B=1, H=8, N=8192, D=128, dtype="bf16", layout="proj"),
        # sixteen such prompts of an odd length: a serving batch's hand-off
        dict(name="handoff 16x32k bf16", op="handoff", B=16, H=8, N=8191, D=128, dtype="bf16", layout="head"),
        # one sequence's token: a handful of heads, latency alone
        dict(name="append 1 fp16 d64", op="append", B=1, H=8, cap=513, D=64, W=100, dtype="fp16", cosine=True),
        # a token of each of 64 sequences
        dict(name="append 64 bf16", op="append", B=64, H=8, cap=1024, D=128, W=128, dtype="bf16", cosine=False),
        # the first tokens after a short prompt, one query head per kv-head
        dict(name="attend 2k fp16 d64", op="attend", B=1, Hq=8, H=8, lo=450, hi=511, cap=513, D=64, W=100, E=100,
             dtype="fp16", mass=True, gaps=False),
        # a token after a 32k-token prompt, four query heads per kv-head
        dict(name="attend 32k bf16", op="attend", B=1, Hq=32, H=8, lo=8192, hi=8192, cap=8448, D=128, W=128, E=128,
             dtype="bf16", mass=True, gaps=False),
        # a batch of prompts of 4k to 32k tokens, every head with its own length, some entries masked
        dict(name="attend 16 ragged bf16", op="attend", B=16, Hq=32, H=8, lo=1024, hi=8192, cap=8448, D=128, W=100,
             E=100, dtype="bf16", mass=True, gaps=True),
        # four 128k-token prompts at one anchor in two: the longest histories, where bandwidth counts
        dict(name="attend 4x128k bf16", op="attend", B=4, Hq=32, H=8, lo=65536, hi=65536, cap=65536, D=128, W=128,
             E=128, dtype="bf16", mass=False, gaps=False),
        # a short history cut by a quarter
        dict(name="evict 2k codes d64", op="evict", B=1, H=8, lo=2048, hi=2048, cap=2048, budget=1536, D=64,
             rows="codes", first=4, recent=128, zeros=0.3),
        # a serving batch's histories cut to a common budget; some are below it and stay
        dict(name="evict 16 ragged codes", op="evict", B=16, H=8, lo=3000, hi=8192, cap=8192, budget=4096, D=128,
             rows="codes", first=4, recent=128, zeros=0.3),
        # a 128k-entry history in 16 bits cut to half, half of its entries never attended: ties at the cut
        dict(name="evict 128k 16-bit", op="evict", B=1, H=8, lo=131072, hi=131072, cap=131072, budget=65536, D=128,
             rows="bf16", first=16, recent=511, zeros=0.6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["handoff", "append", "attend", "attend", "evict"])
    D = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    H = rng.choice([1, 2, 4, 8, 8, 16])
    if op == "handoff":
        N = _log(rng, 1, 60000)
        B = max(1, min(rng.choice([1, 2, 3, 8, 16]), 1000000 // (H * N)))
        return dict(op=op, B=B, H=H, N=N, D=D, dtype=dtype, layout=rng.choice(["head", "proj"]))
    if op == "append":
        return dict(op=op, B=_log(rng, 1, 64), H=min(H, 8), cap=rng.randint(3, 1023), D=D, W=rng.randint(1, 300),
                    dtype=dtype, cosine=rng.random() < 0.5)
    if op == "attend":
        hi = _log(rng, 1, 60000)
        B = max(1, min(_log(rng, 1, 32), 2000000 // (H * hi)))
        lo = rng.choice([hi, hi, hi // 8, 0])
        W = _log(rng, 1, 512)
        G = rng.choice([1, 2, 3, 4, 4, 7, 8, 12])
        return dict(op=op, B=B, Hq=H * G, H=H, lo=lo, hi=hi, cap=hi + rng.randint(0, 300), D=D, W=W,
                    E=rng.choice([W, W, W // 2, 1]), dtype=dtype, mass=rng.random() < 0.6, gaps=rng.random() < 0.4)
    hi = _log(rng, 64, 130000)
    B = max(1, min(_log(rng, 1, 32), 1000000 // (H * hi)))
    budget = max(3, int(hi * rng.uniform(0.3, 0.95)))
    first = rng.randint(0, min(16, budget // 3))
    return dict(op=op, B=B, H=H, lo=rng.choice([hi, hi // 4]), hi=hi, cap=hi + rng.randint(0, 200), budget=budget, D=D,
                rows=rng.choice(["codes", dtype]), first=first, recent=rng.randint(0, min(256, budget // 3)),
                zeros=rng.choice([0.0, 0.3, 0.8]))


# ------------------------------------------------------------------------------------ inputs
def _kv(g, B, H, N, D, dtype, layout="head"):
    """K rows with a constant offset per (head, channel) and V rows, as the layer's projections give them."""
    shape = (B, N, H, D) if layout == "proj" else (B, H, N, D)
    off = torch.randn((1, 1, H, D) if layout == "proj" else (1, H, 1, D), generator=g, device="cuda")
    k = (torch.randn(shape, generator=g, device="cuda") + off).to(dtype)
    v = (torch.randn(shape, generator=g, device="cuda") * 0.5).to(dtype)
    return (k.transpose(1, 2), v.transpose(1, 2)) if layout == "proj" else (k, v)


def _history(g, B, H, cap, D, dtype):
    k, v = _kv(g, B, H, cap, D, dtype)
    return dict(zip(("k_codes", "k_scales", "v_codes", "v_scales"), _quantize(k) + _quantize(v)))


def _lengths(g, case):
    n = torch.randint(case["lo"], case["hi"] + 1, (case["B"], case["H"]), generator=g, device="cuda")
    return n.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, B, H, D = case["op"], case["B"], case["H"], case["D"]
    rand = lambda *s: torch.rand(s, generator=g, device="cuda")  # noqa: E731
    if op == "handoff":
        k, v = _kv(g, B, H, case["N"], D, DTYPES[case["dtype"]], case["layout"])
        return dict(op=op, k=k, v=v)
    cap = case["cap"]
    counts = torch.randint(1, 9, (B, H, cap), generator=g, device="cuda", dtype=torch.int32)
    times = (torch.arange(cap, device="cuda", dtype=torch.int32) * 4).expand(B, H, cap).contiguous()
    if op == "evict":
        # attention weight piles up on few entries; a share of them never drew any
        mass = torch.exp(2 * torch.randn((B, H, cap), generator=g, device="cuda"))
        mass = torch.where(rand(B, H, cap) < case["zeros"], 0.0, mass)
        if case["rows"] == "codes":
            h = _history(g, B, H, cap, D, torch.bfloat16)
            rows = [h["k_codes"], h["k_scales"], h["v_codes"], h["v_scales"], counts, times]
        else:
            rows = [*_kv(g, B, H, cap, D, DTYPES[case["rows"]]), counts, times]
        lengths = _lengths(g, case)
        return dict(op=op, mass=mass, mass0=mass.clone(), lengths=lengths, lengths0=lengths.clone(), rows=rows,
                    budget=case["budget"], first=case["first"], recent=case["recent"])
    dtype, W = DTYPES[case["dtype"]], case["W"]
    s = dict(op=op, hist=_history(g, B, H, cap, D, dtype), counts=counts, times=times)
    s["k_exact"], s["v_exact"] = _kv(g, B, H, W, D, dtype)
    if op == "append":
        n = torch.randint(0, cap, (B, H), generator=g, device="cuda").to(torch.int32)
        e = W + int(seed) % 7  # a full window: its slot e % W leaves
        s["slot"], s["total"] = e % W, e + 4 * cap
        # neighbouring keys: half of the heads' leaving key is near the last anchor's
        near = torch.where(rand(B, H, 1) < 0.5, 0.02, 1.0)
        leaving = s["k_exact"][:, :, s["slot"]].float()
        s["last_key"] = (leaving + near * torch.randn((B, H, D), generator=g, device="cuda")).to(dtype)
        s["k_new"], s["v_new"] = _kv(g, B, H, 1, D, dtype)
        s["state"] = torch.tensor([e, s["total"]], device="cuda", dtype=torch.int64)
        s["cosine"], s["threshold"] = case["cosine"], 0.95 if case["cosine"] else 0.3 * D ** 0.5
        s["lengths"], s["lengths0"] = n, n.clone()
        s["mass"], s["exact_mass"] = rand(B, H, cap), rand(B, H, W)
        return s
    s["lengths"], s["E"] = _lengths(g, case), case["E"]
    if case["gaps"]:  # entries with no tokens behind them draw nothing
        s["counts"] = torch.where(rand(B, H, cap) < 0.06, 0, s["counts"]).to(torch.int32)
    s["q"] = (1.5 * torch.randn((B, case["Hq"], D), generator=g, device="cuda")).to(dtype)
    s["mass"] = rand(B, H, cap) if case["mass"] else None
    s["exact_mass"] = rand(B, H, W) if case["mass"] else None
    return s


# -------------------------------------------------------------------------------- plain forms
def _quantize(x):
    x = x.float()
    B, H, N, D = x.shape
    x = x.reshape(B, H, N, D // 32, 32)
    i = x.amin(-1).view(torch.int32)
    zero = ((i + (i < 0).int() * 0xFFFF) & -0x10000).view(torch.float32)  # rounded down to bf16
    scale = ((x.amax(-1) - zero) / 15).to(torch.bfloat16).float()
    q = ((x - zero[..., None]) / scale[..., None]).round().clamp(0, 15)
    q = torch.where(scale[..., None] == 0, 0.0, q).to(torch.uint8)
    q = q.view(B, H, N, D // 32, 4, 8).transpose(3, 4)
    codes = (q[..., 0::2] | q[..., 1::2] << 4).reshape(B, H, N, D // 2)
    return codes, torch.cat([scale, zero], -1).to(torch.bfloat16)


def _values(codes, scales):
    B, H, N, half = codes.shape
    G = half // 16
    c = codes.view(B, H, N, 4, G, 4)
    c = torch.stack([c & 15, c >> 4], -1).view(B, H, N, 4, G, 8).transpose(3, 4).reshape(B, H, N, G, 32).float()
    s = scales.float()
    return (s[..., G:, None] + s[..., :G, None] * c).view(B, H, N, 2 * half)


def _plain_handoff(s):
    kc, ks = _quantize(s["k"])
    vc, vs = _quantize(s["v"])
    dt = s["k"].dtype
    return dict(k=_values(kc, ks).to(dt), v=_values(vc, vs).to(dt), k_scales=ks, v_scales=vs)


def _plain_append(s):
    h, n, slot = s["hist"], s["lengths"].long(), s["slot"]
    cap = s["counts"].shape[2]
    ke, ve, me = s["k_exact"][:, :, slot], s["v_exact"][:, :, slot], s["exact_mass"][:, :, slot]
    a, b = ke.float(), s["last_key"].float()
    if s["cosine"]:
        near = (a * b).sum(-1) / (((a * a).sum(-1) + 1e-8).sqrt() * ((b * b).sum(-1) + 1e-8).sqrt()) >= s["threshold"]
    else:
        near = ((a - b) ** 2).sum(-1) <= s["threshold"] ** 2
    merge = near & (n > 0)
    add = ~merge & (n < cap)
    last, at = (n - 1).clamp(min=0)[..., None], n.clamp(max=cap - 1)[..., None]

    def put(buf, rows):  # rows of the heads that append, at their length
        i = at.view(*at.shape, *([1] * (buf.dim() - 3))).expand(-1, -1, -1, *buf.shape[3:])
        rows = rows.reshape(i.shape).to(buf.dtype)
        buf.scatter_(2, i, torch.where(add.view(*add.shape, *([1] * (buf.dim() - 2))), rows, buf.gather(2, i)))

    s["counts"].scatter_add_(2, last, merge[..., None].int())
    s["mass"].scatter_add_(2, last, torch.where(merge, me, 0.0)[..., None])
    for name, x in (("k", ke), ("v", ve)):
        codes, scales = _quantize(x[:, :, None])
        put(h[name + "_codes"], codes)
        put(h[name + "_scales"], scales)
    put(s["counts"], torch.ones_like(n))
    put(s["times"], torch.full_like(n, s["total"] - s["k_exact"].shape[2]))
    put(s["mass"], me)
    s["last_key"].copy_(torch.where(add[..., None], ke, s["last_key"]))
    s["lengths"].add_(add.int())
    s["k_exact"][:, :, slot] = s["k_new"][:, :, 0]
    s["v_exact"][:, :, slot] = s["v_new"][:, :, 0]
    s["exact_mass"][:, :, slot] = 0


def _plain_attend(s):
    h, q, E = s["hist"], s["q"], s["E"]
    B, H, cap = s["counts"].shape
    D = q.shape[-1]
    q = q.float().view(B, H, -1, D)
    live = torch.arange(cap, device=q.device) < s["lengths"][..., None]
    live = (live & (s["counts"] > 0))[:, :, None]
    c = s["counts"][:, :, None].float()
    sp = q @ _values(h["k_codes"], h["k_scales"]).transpose(2, 3) * D ** -0.5
    sp = torch.where(live, sp + torch.where(live, c, 1.0).log(), -math.inf)
    se = q @ s["k_exact"][:, :, :E].float().transpose(2, 3) * D ** -0.5
    m = torch.cat([sp, se], -1).amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    wp, we = (sp - m).exp(), (se - m).exp()
    l = wp.sum(-1, keepdim=True) + we.sum(-1, keepdim=True)
    l = torch.where(l == 0, 1.0, l)
    wp, we = wp / l, we / l
    v = torch.where(live[:, :, 0, :, None], _values(h["v_codes"], h["v_scales"]), 0.0)
    o = wp @ v + we @ s["v_exact"][:, :, :E].float()
    if s["mass"] is not None:
        s["mass"].add_(wp.sum(2))
        s["exact_mass"][:, :, :E].add_(we.sum(2))
    return o.view(B, -1, D).to(s["q"].dtype)


def _plain_evict(s):
    mass, n, budget = s["mass"], s["lengths"].long()[..., None], s["budget"]
    B, H, cap = mass.shape
    i = torch.arange(cap, device=mass.device)
    key = torch.where((i < s["first"]) | (i >= n - s["recent"]), math.inf, mass)
    key = torch.where(i < n, key, -math.inf)
    rank = key.sort(dim=-1, descending=True, stable=True).indices.argsort(-1)
    cut = n > budget
    keep = torch.where(cut, (rank < budget) & (i < n), i < n)
    src = (~keep).int().sort(dim=-1, stable=True).indices[..., :budget]
    src = torch.where(cut, src, i[:budget])
    for buf in (mass, *s["rows"]):
        j = src.view(*src.shape, *([1] * (buf.dim() - 3))).expand(-1, -1, -1, *buf.shape[3:])
        buf[:, :, :budget] = buf.gather(2, j)
    s["lengths"].clamp_(max=budget)


# --------------------------------------------------------------------------------- the passes
def run(s):
    if own:
        from deltaattention_b200 import ops
    op = s["op"]
    if op == "handoff":
        if not own:
            return _plain_handoff(s)
        h = ops.kv4_quantize(s["k"], s["v"])
        k, v = ops.kv4_dequantize(h, s["k"].dtype)
        return dict(k=k, v=v, k_scales=h.k_scales, v_scales=h.v_scales)
    if op == "append":
        # back to the same lengths, so that every pass appends or merges one token
        s["lengths"].copy_(s["lengths0"])
        if own:
            ops.decode_update_kv4(s["k_new"], s["v_new"], ops.KV4(**s["hist"]), s["counts"], s["times"], s["lengths"],
                                  s["last_key"], s["k_exact"], s["v_exact"], s["state"], threshold=s["threshold"],
                                  similarity="cosine" if s["cosine"] else "euclidean", mass=s["mass"],
                                  exact_mass=s["exact_mass"])
        else:
            _plain_append(s)
        # the codes come as bytes of two, and have to be equal
        return {**s["hist"], **{k: s[k] for k in ("counts", "times", "lengths", "last_key", "k_exact", "v_exact",
                                                  "mass", "exact_mass")}}
    if op == "attend":
        if own:
            out = ops.decode_attention_kv4(s["q"], ops.KV4(**s["hist"]), s["counts"], s["lengths"], s["k_exact"],
                                           s["v_exact"], exact_len=s["E"], mass=s["mass"], exact_mass=s["exact_mass"])
        else:
            out = _plain_attend(s)
        return dict(out=out, mass=s["mass"], exact_mass=s["exact_mass"])
    # back to the same lengths and weights, so that every pass selects and moves the same entries
    s["lengths"].copy_(s["lengths0"])
    s["mass"].copy_(s["mass0"])
    if own:
        ops.evict_by_mass(s["mass"], s["lengths"], s["rows"], s["budget"], keep_first=s["first"],
                          keep_recent=s["recent"])
    else:
        _plain_evict(s)
    # rows are moved as they are; those in 4 bits come as bytes of two codes, and have to be equal
    return dict(mass=s["mass"], lengths=s["lengths"], rows=s["rows"])


def work(case):
    op, B, H, D = case["op"], case["B"], case["H"], case["D"]
    row = D // 2 + D // 8  # one row's codes and scales, bytes
    if op == "handoff":  # K and V: values in, codes out and in, values out
        n = B * H * case["N"]
        return dict(bytes=2 * n * (4 * D + 2 * row), flops=2 * n * D * 8)
    if op == "append":  # new and leaving token, last key, the appended row, ring slots
        return dict(bytes=B * H * (2 * D * 2 * 3 + 2 * D * 2 + 2 * row + 40), flops=B * H * D * 20)
    n = B * H * (case["lo"] + case["hi"]) / 2
    if op == "attend":
        e = B * H * case["E"]
        b = n * (2 * row + 4) + e * 4 * D + 2 * B * case["Hq"] * D * 2
        if case["mass"]:
            b += 8 * (n + e)
        return dict(bytes=b, flops=4 * (n + e) * D * case["Hq"] // H)
    width = 2 * (row if case["rows"] == "codes" else 2 * D) + 8 + 4
    kept = B * H * min(case["budget"], (case["lo"] + case["hi"]) / 2)
    return dict(bytes=4 * n + 2 * kept * width, flops=n)


# -------------------------------------------------------------------------------- in 64 bits
def _exact_bf16(x, down=False):
    m, e = torch.frexp(x)
    m = m * 256
    return torch.ldexp((m.floor() if down else m.round()) / 256, e)


def _exact_quantize(x):
    """(value of every element, scales then zeros) of rows x, in 64 bits."""
    x = x.double()
    g = x.unflatten(-1, (-1, 32))
    zero = _exact_bf16(g.min(-1).values, down=True)
    scale = _exact_bf16((g.max(-1).values - zero) / 15.0)
    step = torch.where(scale == 0, 1.0, scale)[..., None]
    code = torch.clamp(torch.round((g - zero[..., None]) / step), 0, 15)
    return (zero[..., None] + scale[..., None] * code).flatten(-2), torch.cat([scale, zero], -1)


def _exact_values(codes, scales):
    D = codes.shape[-1] * 2
    d = torch.arange(D, device=codes.device)
    word = (d % 32) // 8 * (D // 32) + d // 32
    byte, high = word * 4 + d % 8 // 2, d % 2
    c = (codes[..., byte].long() >> (4 * high)) % 16
    s = scales.double()
    return s[..., D // 32 + d // 32] + s[..., d // 32] * c


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "handoff":
        out = {}
        for x in ("k", "v"):
            parts = [_exact_quantize(s[x][b]) for b in range(s[x].shape[0])]
            out[x] = torch.stack([p[0] for p in parts])
            out[x + "_scales"] = torch.stack([p[1] for p in parts])
        return out
    if op == "append":
        B, H, cap = s["counts"].shape
        slot = s["slot"]
        out = {k: s["hist"][k].double() for k in ("k_scales", "v_scales")}
        out |= {k: s[k].double() for k in ("last_key", "k_exact", "v_exact", "mass", "exact_mass")}
        lens = s["lengths"].tolist()
        for b in range(B):
            for h in range(H):
                n, x, y = lens[b][h], s["k_exact"][b, h, slot].double(), s["last_key"][b, h].double()
                if s["cosine"]:
                    near = x.dot(y) / ((x.dot(x) + 1e-8).sqrt() * (y.dot(y) + 1e-8).sqrt()) >= s["threshold"]
                else:
                    near = (x - y).dot(x - y) <= s["threshold"] ** 2
                if n > 0 and bool(near):
                    out["mass"][b, h, n - 1] += s["exact_mass"][b, h, slot].double()
                elif n < cap:
                    out["mass"][b, h, n] = s["exact_mass"][b, h, slot].double()
                    out["last_key"][b, h] = x
                    for c in ("k", "v"):
                        out[c + "_scales"][b, h, n] = _exact_quantize(s[c + "_exact"][b, h, slot])[1]
        for c in ("k", "v"):
            out[c + "_exact"][:, :, slot] = s[c + "_new"][:, :, 0].double()
        out["exact_mass"][:, :, slot] = 0
        return out
    if op == "attend":
        B, H, cap = s["counts"].shape
        D, E = s["q"].shape[-1], s["E"]
        G = s["q"].shape[1] // H
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        mass = None if s["mass"] is None else s["mass"].double()
        emass = None if s["mass"] is None else s["exact_mass"].double()
        lens = s["lengths"].tolist()
        for b in range(B):
            for h in range(H):
                at = torch.nonzero(s["counts"][b, h, :lens[b][h]] > 0)[:, 0]
                part = {k: v[b, h, at] for k, v in s["hist"].items()}
                k = torch.cat([_exact_values(part["k_codes"], part["k_scales"]), s["k_exact"][b, h, :E].double()])
                v = torch.cat([_exact_values(part["v_codes"], part["v_scales"]), s["v_exact"][b, h, :E].double()])
                if not len(k):
                    continue
                c = torch.cat([s["counts"][b, h, at].double(), torch.ones(E, dtype=torch.float64, device="cuda")])
                z = (k @ s["q"][b, h * G:(h + 1) * G].double().T) / math.sqrt(D)
                w = c[:, None] * torch.exp(z - z.max(0).values)
                w = w / w.sum(0)
                out[b, h * G:(h + 1) * G] = w.T @ v
                if mass is not None:
                    mass[b, h].index_add_(0, at, w[:len(at)].sum(1))
                    emass[b, h, :E] += w[len(at):].sum(1)
        return dict(out=out, mass=mass, exact_mass=emass)
    mass = s["mass"].double().cpu().numpy()
    rows = [r.double() if r.is_floating_point() else None for r in s["rows"]]
    done = torch.from_numpy(mass.copy())
    for b in range(mass.shape[0]):
        for h, n in enumerate(s["lengths"][b].tolist()):
            if n <= s["budget"]:
                continue
            first, end = s["first"], n - s["recent"]
            most = s["budget"] - first - s["recent"]
            middle = sorted(range(first, end), key=lambda i: (-mass[b, h, i], i))[:most]
            kept = torch.tensor([*range(first), *sorted(middle), *range(end, n)])
            done[b, h, :len(kept)] = torch.from_numpy(mass[b, h])[kept]
            for r in rows:
                if r is not None:
                    r[b, h, :len(kept)] = r[b, h, kept.to(r.device)]
    return dict(mass=done, lengths=None, rows=rows)
