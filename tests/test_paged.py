"""Paged key / value cache: append with rotation, attention of packed prompts, of prompts over the pages, and decode
with shared prefixes, against plain implementations in 64 bits.

Tolerances, from the formulas:
* a rotated element is x cos + y sin in fp32 and rounded once: the type's unit roundoff u of it (2^-8 bf16,
  2^-11 fp16) and fp32's rounding of the two products;
* attention: weights p are held in 16 bits with 32-bit sums, so an output is off by u * sum(p |v|) at most for
  the weights and u of itself for its own rounding; scores are 32-bit dot products of terms that sum to
  some tens, off by 2^-14 of a weight at most. 2 u * max|v| + 2^-13 * max|v| covers all of them.
"""
import math

import pytest
import torch

from deltaattention_b200 import _lib as L

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from deltaattention_b200 import ops as o
    L.load()
    return o


@pytest.fixture(autouse=True)
def no_device_errors(request):
    yield
    if "gpu" in request.keywords and torch.cuda.is_available():
        assert not any(L.workspace_errors())


# ------------------------------------------------------------------ plain forms in 64 bits
def rotate64(x, cos, sin):
    """x [n, H, D] with tables [n, D]."""
    h = x.shape[-1] // 2
    turned = torch.cat([-x[..., h:], x[..., :h]], -1)
    return x * cos[:, None] + turned * sin[:, None]


def attend64(q, k, v, see, scale):
    """q [n, Hq, D], k / v [L, H, D]; query i sees the first see[i] rows."""
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    n, Hq, D = q.shape
    G = Hq // k.shape[1]
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    for i in range(n):
        m = int(see[i])
        if m <= 0:
            continue
        for h in range(k.shape[1]):
            w = torch.softmax(q[i, h * G:(h + 1) * G] @ k[:m, h].T * scale, -1)
            out[i, h * G:(h + 1) * G] = w @ v[:m, h]
    return out


def check(out, ref, v):
    u = UNIT[out.dtype]
    tol = (2 * u + 2.0 ** -13) * v.float().abs().max().item()
    err = (out.cpu().double() - ref).abs().max().item() if out.numel() else 0.0
    assert err <= tol, (err, tol)


class Pool:
    """A pool filled everywhere, and the rows of its sequences as they should be."""

    def __init__(self, ops, B, H, D, ps, lens, dt, seed, layout="head", spare=2, share=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.ps = lens, ps
        mp = max(1, share // ps, max(-(-n // ps) for n in lens)) + spare
        first = share // ps
        P = first + B * mp + 1
        shape = (P, ps, H, D) if layout == "row" else (P, H, ps, D)
        k = torch.randn(shape, generator=g) + torch.randn(1, generator=g)
        v = torch.randn(shape, generator=g)
        self.k, self.v = (t.to(DT[dt]).cuda() for t in (k, v))
        if layout == "row":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        order = torch.randperm(P, generator=g)
        table = order[:B * mp].view(B, mp).clone()
        if first:
            table[:, :first] = order[B * mp:B * mp + first]
        self.table = table.to(torch.int32).cuda()
        self.lengths = torch.tensor(lens, dtype=torch.int32).cuda()
        self.kv = ops.PagedKV(self.k, self.v)

    def rows(self, b, n=None):
        """K and V rows [n, H, D] of a sequence."""
        n = self.lens[b] if n is None else n
        p = torch.arange(n)
        page, row = self.table[b].cpu().long()[p // self.ps], p % self.ps
        return self.k.cpu()[page, :, row], self.v.cpu()[page, :, row]


def starts(n, device="cuda"):
    return torch.tensor([0, *n]).cumsum(0).to(torch.int32).to(device)


# -------------------------------------------------------------------------------------- append
@gpu
@pytest.mark.parametrize("news,pasts,Hq,H,D,ps,dt,tables,layout,fused", [
    ([1], [0], 8, 8, 64, 16, "fp16", "fp16", "head", False),
    ([1, 1, 1], [5, 0, 31], 12, 3, 128, 32, "bf16", "fp32", "row", True),
    ([17, 0, 1, 130], [3, 9, 0, 64], 4, 2, 128, 64, "bf16", "bf16", "head", True),
    ([200, 33], [0, 0], 7, 1, 64, 16, "bf16", "fp32", "row", True),
    ([5] * 40, [0] * 40, 3, 3, 64, 128, "fp16", "fp32", "head", False),
    ([2] * 1100, [1] * 1100, 2, 1, 64, 16, "fp16", "fp32", "head", False),
    ([700], [900], 32, 8, 128, 256, "fp16", "fp16", "row", True)])
def test_append(ops, news, pasts, Hq, H, D, ps, dt, tables, layout, fused):
    B, T = len(news), sum(news)
    pool = Pool(ops, B, H, D, ps, [a + b for a, b in zip(news, pasts)], dt, 7, layout)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T + 3, (Hq + 2 * H) * D, generator=g).to(DT[dt]).cuda()
    q, k, v = (t.unflatten(1, (-1, D)) for t in x.split([Hq * D, H * D, H * D], 1))
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    n = max(pool.lens)
    ang = torch.arange(n)[:, None].double() * 1e4 ** (-torch.arange(0, D, 2).double() / D)
    ang = torch.cat([ang, ang + 0.1], 1)  # the halves of the tables need not agree
    td = torch.float32 if tables == "fp32" else DT[dt]
    cos, sin = ang.cos().to(td).cuda(), ang.sin().to(td).cuda()
    one = all(x == 1 for x in news)
    before = pool.k.clone(), pool.v.clone()
    q_out = torch.full((T + 3, Hq, D), 7.0, dtype=DT[dt], device="cuda")
    if one:
        x, q, k, v, q_out = x[:T], q[:T], k[:T], v[:T], q_out[:T]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.paged_append(k, v, pool.kv, pool.table, pool.lengths, cu_seqlens=None if one else starts(news),
                           cos=cos[None], sin=sin[None], q=q, q_out=q_out, err=err)
    assert got is q_out and int(err) == 0
    touched = torch.zeros(pool.k.shape[0], ps, dtype=torch.bool)
    at, u = 0, UNIT[DT[dt]]
    kc, vc = pool.k.cpu(), pool.v.cpu()
    for b in range(B):
        p = torch.arange(pasts[b], pool.lens[b])
        page, row = pool.table[b].cpu().long()[p // ps], p % ps
        touched[page, row] = True
        c, s = cos.cpu().double()[p], sin.cpu().double()[p]
        for x, y in ((k, kc[page, :, row]), (q, q_out[at:at + news[b]].cpu())):
            x = x[at:at + news[b]].cpu().double()
            ref = rotate64(x, c, s)
            tol = u * ref.abs() + 2.0 ** -22 * (x.abs().amax(-1, keepdim=True) if len(x) else x[..., :1])
            assert ((y.double() - ref).abs() <= tol).all()
        assert torch.equal(vc[page, :, row], v[at:at + news[b]].cpu())
        at += news[b]
    # every other row of the pool and of q_out is as it was
    for x, y in zip(before, (kc, vc)):
        assert torch.equal(x.cpu().transpose(1, 2)[~touched], y.transpose(1, 2)[~touched])
    assert (q_out[T:] == 7).all()


@gpu
def test_append_without_rotation_and_idle_places(ops):
    pool = Pool(ops, 3, 2, 64, 16, [4, 0, 20], "bf16", 1)
    k = torch.randn(3, 2, 64).bfloat16().cuda()
    v = torch.randn(3, 2, 64).bfloat16().cuda()
    before = pool.k.clone()
    assert ops.paged_append(k, v, pool.kv, pool.table, pool.lengths) is None
    for b, n in ((0, 4), (2, 20)):
        kr, vr = pool.rows(b)
        assert torch.equal(kr[n - 1], k[b].cpu()) and torch.equal(vr[n - 1], v[b].cpu())
    assert int((pool.k != before).any(-1).any(1).sum()) == 2


@gpu
def test_append_in_place_and_wrong_contents(ops):
    """q may be rotated in place; page numbers, lengths and positions out of range store nothing and say so."""
    pool = Pool(ops, 2, 1, 64, 16, [20, 9], "fp16", 2, spare=0)
    k = torch.randn(2, 1, 64).half().cuda()
    q = torch.randn(2, 4, 64).half().cuda()
    cos = torch.randn(32, 64).cuda()
    sin = torch.randn(32, 64).cuda()
    other = ops.paged_append(k, k, pool.kv, pool.table, pool.lengths, cos=cos, sin=sin, q=q)
    same = ops.paged_append(k, k, pool.kv, pool.table, pool.lengths, cos=cos, sin=sin, q=q, q_out=q)
    assert same is q and torch.equal(q, other)
    before = pool.k.clone()
    k2 = k + 1
    for bad, n, rows, code in ((pool.k.shape[0], 20, 32, 0x601), (-1, 20, 32, 0x601), (0, 33, 64, 0x602), (0, 20, 19, 0x603)):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        table = pool.table.clone()
        table[0, 1] = bad
        lengths = torch.tensor([n, 0], dtype=torch.int32, device="cuda")
        tabs = torch.zeros(rows, 64, device="cuda")
        ops.paged_append(k2, k2, pool.kv, table, lengths, cos=tabs, sin=tabs, err=err)
        assert int(err) == code
        assert torch.equal(before, pool.k)


# ------------------------------------------------------------------------------ packed prompts
LENS = [([1], 1, 1, 64), ([500], 8, 8, 64), ([128], 4, 4, 128), ([129, 1, 127], 8, 2, 128), ([0, 300, 0, 65], 4, 1, 64),
        ([33, 257, 64], 6, 2, 128), ([40, 41], 14, 2, 64), ([70] * 5, 12, 1, 128), ([300], 5, 1, 128), ([9, 200], 128, 1, 64)]


def prompt_inputs(n, Hq, H, D, dt, fused=True, spare=3):
    g = torch.Generator().manual_seed(sum(n) * Hq + D)
    x = torch.randn(sum(n) + spare, (Hq + 2 * H) * D, generator=g).to(DT[dt]).cuda()
    q, k, v = (t.unflatten(1, (-1, D)) for t in x.split([Hq * D, H * D, H * D], 1))
    return (q, k, v) if fused else (q.contiguous(), k.contiguous(), v.contiguous())


@gpu
@pytest.mark.parametrize("dt,causal,fused", [("bf16", True, True), ("fp16", True, False), ("bf16", False, False)])
@pytest.mark.parametrize("n,Hq,H,D", LENS)
def test_prompts(ops, n, Hq, H, D, dt, causal, fused):
    q, k, v = prompt_inputs(n, Hq, H, D, dt, fused)
    q = q * 2
    T = sum(n)
    out = torch.full((T + 3, Hq, D), 7.0, dtype=DT[dt], device="cuda")
    got = ops.flash_varlen(q, k, v, starts(n), causal=causal, out=out)
    assert got is out
    at = 0
    for m in n:
        s = slice(at, at + m)
        see = torch.arange(1, m + 1) if causal else torch.full((m,), m)
        check(out[s], attend64(q[s], k[s], v[s], see, D ** -0.5), v)
        at += m
    assert (out[T:] == 7).all()  # tokens behind the last sequence


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_prompts_with_rising_scores(ops, dt):
    """Scores that grow along the keys move the running maximum in every tile, by a little and by a lot."""
    n, Hq, H, D = [700], 4, 2, 64
    q, k, v = prompt_inputs(n, Hq, H, D, dt, False, 0)
    for step in (0.002, 0.05, -0.05):
        kk = (k.float() * 0.1 + step * torch.arange(700, device="cuda")[:, None, None]).to(DT[dt])
        qq = (q.float() * 0.1 + 1).to(DT[dt])
        out = ops.flash_varlen(qq, kk, v, starts(n))
        ref = attend64(qq, kk, v, torch.arange(1, 701), D ** -0.5)
        # scores of up to 280 in 32-bit sums of 64 terms: off by 2^-24 * 280 * 8 at most, 2^-13 of a weight
        check(out, ref, v)


@gpu
def test_prompts_ignore_what_lies_behind_them(ops):
    """NaN and infinities in the next sequence's rows and in tokens behind the last one reach nobody else."""
    n, Hq, H, D = [100, 60, 130], 4, 2, 128
    q, k, v = prompt_inputs(n, Hq, H, D, "bf16", False)
    ref = ops.flash_varlen(q, k, v, starts(n))
    for t in (q, k, v):
        t[100:160] = float("nan")
        t[290:] = float("inf")
    out = ops.flash_varlen(q, k, v, starts(n))
    assert torch.equal(out[:100], ref[:100]) and torch.equal(out[160:290], ref[160:290])
    assert out[100:160].isnan().all()


@gpu
def test_prompts_scale(ops):
    n, Hq, H, D = [50], 2, 2, 64
    q, k, v = prompt_inputs(n, Hq, H, D, "fp16", False, 0)
    out = ops.flash_varlen(q, k, v, starts(n), sm_scale=0.3)
    check(out, attend64(q, k, v, torch.arange(1, 51), 0.3), v)
    for scale in (0.0, -0.2, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="sm_scale"):
            ops.flash_varlen(q, k, v, starts(n), sm_scale=scale)


# ------------------------------------------------------------------------ prompts over the pages
@gpu
@pytest.mark.parametrize("news,pasts,Hq,H,D,ps,dt,layout", [
    ([1], [0], 1, 1, 64, 16, "fp16", "head"), ([300], [700], 16, 4, 64, 32, "fp16", "row"),
    ([40, 0, 3, 129], [500, 77, 0, 128], 8, 2, 128, 16, "bf16", "head"), ([64, 200], [0, 0], 7, 1, 128, 64, "bf16", "row"),
    ([100, 90], [900, 33], 4, 4, 128, 128, "bf16", "head"), ([130], [600], 12, 2, 64, 256, "bf16", "row"),
    ([10, 20, 30], [2000, 10, 1000], 6, 2, 128, 16, "fp16", "head")])
def test_prompts_over_pages(ops, news, pasts, Hq, H, D, ps, dt, layout):
    pool = Pool(ops, len(news), H, D, ps, [a + b for a, b in zip(news, pasts)], dt, 11, layout)
    T = sum(news)
    g = torch.Generator().manual_seed(T)
    q = (2 * torch.randn(T + 2, Hq, D, generator=g)).to(DT[dt]).cuda()
    for causal in (True, False):
        out = torch.full_like(q, 7.0)
        ops.flash_paged(q, pool.kv, pool.table, pool.lengths, starts(news), causal=causal, out=out)
        at = 0
        for b, m in enumerate(news):
            k, v = pool.rows(b)
            see = pasts[b] + torch.arange(1, m + 1) if causal else torch.full((m,), pool.lens[b])
            check(out[at:at + m], attend64(q[at:at + m], k, v, see, D ** -0.5), pool.v)
            at += m
        assert (out[T:] == 7).all()


@gpu
def test_pages_hold_anything_past_the_length(ops):
    """Stale rows of a sequence's last page and stale page numbers past it are not looked at."""
    news, pasts = [5, 140], [6, 3]
    pool = Pool(ops, 2, 2, 64, 32, [11, 143], "bf16", 3)
    q = torch.randn(145, 4, 64).bfloat16().cuda()
    d = torch.randn(2, 4, 64).bfloat16().cuda()
    ref = ops.flash_paged(q, pool.kv, pool.table, pool.lengths, starts(news))
    dref = ops.decode_attention_paged(d, pool.kv, pool.table, pool.lengths)
    keep = torch.zeros(pool.k.shape[0], 32, dtype=torch.bool)
    for b, n in enumerate(pool.lens):
        p = torch.arange(n)
        keep[pool.table[b].cpu().long()[p // 32], p % 32] = True
        pool.table[b, -(-n // 32):] = 10 ** 9
    for t in (pool.k, pool.v):
        t.transpose(1, 2)[~keep.cuda()] = float("nan")
    assert torch.equal(ops.flash_paged(q, pool.kv, pool.table, pool.lengths, starts(news)), ref)
    assert torch.equal(ops.decode_attention_paged(d, pool.kv, pool.table, pool.lengths), dref)


@gpu
def test_queries_before_the_first_row(ops):
    """More queries than rows: those at negative positions give 0."""
    pool = Pool(ops, 2, 1, 64, 16, [3, 0], "fp16", 4)
    q = torch.randn(7, 2, 64).half().cuda()
    out = ops.flash_paged(q, pool.kv, pool.table, pool.lengths, starts([5, 2]))
    k, v = pool.rows(0)
    check(out[:5], attend64(q[:5], k, v, [-1, 0, 1, 2, 3], 64 ** -0.5), v)
    assert (out[:2] == 0).all() and (out[5:] == 0).all()
    assert (ops.flash_paged(q, pool.kv, pool.table, pool.lengths, starts([5, 2]), causal=False)[5:] == 0).all()


# -------------------------------------------------------------------------------------- decode
@gpu
@pytest.mark.parametrize("lens,share,cu,Hq,H,D,ps,dt,layout", [
    ([1], 0, None, 1, 1, 64, 16, "fp16", "head"),
    ([1900], 0, None, 16, 4, 64, 16, "fp16", "head"),
    ([128, 0, 129, 5], 0, None, 8, 2, 128, 32, "bf16", "row"),
    ([3000, 10, 700], 0, None, 32, 8, 128, 64, "bf16", "head"),
    ([600, 601, 999, 512], 512, [0, 4], 8, 2, 128, 16, "bf16", "head"),
    ([600, 601, 999, 512, 40], 512, [0, 4], 7, 1, 128, 64, "bf16", "row"),
    ([300] * 3 + [0] + [290] * 3, 256, [0, 3, 7], 4, 4, 64, 128, "fp16", "head"),
    ([300 + 7 * i for i in range(70)], 288, [0, 70], 16, 2, 64, 32, "bf16", "row"),
    ([200 + i for i in range(40)], 192, [0, 1, 1, 33], 12, 2, 128, 16, "fp16", "head"),
    ([0, 0], 64, [0, 2], 2, 1, 64, 16, "bf16", "head")])
def test_decode(ops, lens, share, cu, Hq, H, D, ps, dt, layout):
    pool = Pool(ops, len(lens), H, D, ps, lens, dt, 5, layout, share=share)
    if share:  # the sequences outside the groups and those shorter than the prefix share too: harmless
        assert share % ps == 0
    g = torch.Generator().manual_seed(len(lens))
    q = (2 * torch.randn(len(lens), Hq, D, generator=g)).to(DT[dt]).cuda()
    kw = {}
    if cu is not None:
        kw = dict(prefix_cu=torch.tensor(cu, dtype=torch.int32).cuda(),
                  prefix_lengths=torch.full((len(cu) - 1,), share, dtype=torch.int32).cuda())
    out = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, **kw)
    for b, n in enumerate(lens):
        k, v = pool.rows(b)
        check(out[b:b + 1], attend64(q[b:b + 1], k, v, [n], D ** -0.5), pool.v)
    if share:  # part of a page, and more than a member has
        for n in (share - 5, share + 9, 1):
            kw["prefix_lengths"].fill_(n)
            first = lens[:cu[-1]]
            if n > share and any(x > share for x in first):
                continue  # the rows past the shared pages differ
            out = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, **kw)
            for b, m in enumerate(lens):
                k, v = pool.rows(b)
                check(out[b:b + 1], attend64(q[b:b + 1], k, v, [m], D ** -0.5), pool.v)


# ------------------------------------------------------------------------------------ refusals
def test_refuses_cpu_tensors():
    from deltaattention_b200 import ops
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    pool = ops.PagedKV.empty(2, 1, 16, 64, torch.bfloat16, "cpu")
    t, n = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for call in (lambda: ops.paged_append(x, x, pool, t, n), lambda: ops.flash_varlen(x, x, x, n),
                 lambda: ops.flash_paged(x, pool, t, n, n), lambda: ops.decode_attention_paged(x, pool, t, n)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_library_refuses_bad_sizes():
    """The C entries check sizes and alignment before any CUDA call."""
    lib = L.load()
    s = L.strides([64] * 13)
    def append(D=64, ps=16, heads=1, tokens=2, batch=2, mp=1, k=64, table=64, cos=None, sin=None, q=None, qo=None, qh=0):
        return lib.dab_paged_append(k, 64, q, qo, 64, 64, table, 64, None, cos, sin, s, 2, 0, tokens, batch, heads, qh, D, 4, ps,
                                    mp, 9, None, None)
    for kw, text in ((dict(D=96), "head_dim"), (dict(ps=24), "page_size"), (dict(ps=512), "page_size"), (dict(heads=0), "head"),
                     (dict(tokens=3), "sizes"), (dict(mp=1 << 27), "rows"), (dict(k=None), "null"), (dict(k=72), "16-byte"),
                     (dict(table=None), "null"), (dict(cos=64), "null"), (dict(q=64, qo=64, qh=1), "rotation tables")):
        assert append(**kw) != 0
        assert text in lib.dab_last_error().decode(), kw
    def varlen(D=64, G=1, H=1, q=64, ws=64, nb=1 << 40):
        return lib.dab_flash_varlen(q, 64, 64, 64, 64, s, 1.0, 1, 2, 5, 1, H, G, D, ws, nb, None)
    for kw, text in ((dict(D=32), "head_dim"), (dict(G=129), "128 q-heads"), (dict(H=0), "q-heads"), (dict(q=None), "null"),
                     (dict(q=8), "16-byte"), (dict(ws=None), "workspace"), (dict(nb=1), "workspace"), (dict(ws=8), "aligned")):
        assert varlen(**kw) != 0
        assert text in lib.dab_last_error().decode(), kw
    def decode(groups=0, cu=None, ps=16):
        return lib.dab_decode_attention_paged(64, 64, 64, 64, 64, 64, cu, cu, s, 1.0, 2, 3, 1, 1, 64, 4, ps, 2, groups, 64,
                                              1 << 40, None)
    for kw, text in ((dict(groups=4, cu=64), "group"), (dict(groups=1), "prefix_cu"), (dict(ps=8), "page_size")):
        assert decode(**kw) != 0
        assert text in lib.dab_last_error().decode(), kw


@gpu
def test_refusals(ops):
    pool = Pool(ops, 2, 2, 64, 16, [20, 5], "bf16", 6)
    kv, table, n = pool.kv, pool.table, pool.lengths
    q, k = torch.zeros(2, 4, 64).bfloat16().cuda(), torch.zeros(2, 2, 64).bfloat16().cuda()
    tab = torch.zeros(30, 64).cuda()
    cu = starts([1, 1])
    bad = [
        (TypeError, lambda: ops.paged_append(k.half(), k, kv, table, n)),
        (ValueError, lambda: ops.paged_append(k, k[:1], kv, table, n)),
        (ValueError, lambda: ops.paged_append(k[:1], k[:1], kv, table, n)),
        (ValueError, lambda: ops.paged_append(k, k, kv, table.long(), n)),
        (ValueError, lambda: ops.paged_append(k, k, kv, table, n.long())),
        (ValueError, lambda: ops.paged_append(k, k, kv, table, n[:1])),
        (ValueError, lambda: ops.paged_append(k, k, kv, table, n, cos=tab)),
        (ValueError, lambda: ops.paged_append(k, k, kv, table, n, q=q)),
        (ValueError, lambda: ops.paged_append(k, k, kv, table, n, cos=tab, sin=tab, q_out=q)),
        (ValueError, lambda: ops.paged_append(k, k, kv, table, n, cos=tab[:, :32], sin=tab[:, :32])),
        (TypeError, lambda: ops.paged_append(k, k, kv, table, n, cos=tab.half(), sin=tab.half())),
        (ValueError, lambda: ops.paged_append(k, k, kv, table, n, cos=tab, sin=tab, q=q, q_out=q[:1].expand(2, 4, 64))),
        (ValueError, lambda: ops.paged_append(k, k, ops.PagedKV(kv.k, kv.v.contiguous()[:, :1]), table, n)),
        (ValueError, lambda: ops.paged_append(k, k, ops.PagedKV(kv.k[:, :, :8], kv.v[:, :, :8]), table, n)),
        (ValueError, lambda: ops.paged_append(torch.zeros(2, 2, 72).bfloat16().cuda()[..., 1:65], k, kv, table, n)),
        (ValueError, lambda: ops.flash_varlen(q, k, k, cu.long())),
        (ValueError, lambda: ops.flash_varlen(q, k[:1], k, cu)),
        (ValueError, lambda: ops.flash_varlen(q[:, :3], k, k, cu)),
        (TypeError, lambda: ops.flash_varlen(q.float(), k.float(), k.float(), cu)),
        (TypeError, lambda: ops.flash_varlen(q, k.half(), k, cu)),
        (ValueError, lambda: ops.flash_varlen(q, k, k, cu, out=q[:1].expand(2, 4, 64))),
        (ValueError, lambda: ops.flash_varlen(q, k, k, cu, workspace=torch.zeros(1 << 20).cuda())),
        (RuntimeError, lambda: ops.flash_varlen(q, k, k, cu, workspace=torch.zeros(16, dtype=torch.uint8).cuda())),
        (ValueError, lambda: ops.flash_paged(q, kv, table, n, cu[:2])),
        (TypeError, lambda: ops.flash_paged(q.half(), kv, table, n, cu)),
        (ValueError, lambda: ops.decode_attention_paged(q[:1], kv, table, n)),
        (ValueError, lambda: ops.decode_attention_paged(q, kv, table, n, prefix_cu=cu)),
        (ValueError, lambda: ops.decode_attention_paged(q, kv, table, n, prefix_cu=cu[:2], prefix_lengths=n)),
        (ValueError, lambda: ops.decode_attention_paged(q, kv, table, n, prefix_cu=starts([1, 1, 0]),
                                                        prefix_lengths=torch.zeros(3, dtype=torch.int32).cuda())),
        (RuntimeError, lambda: ops.decode_attention_paged(q, kv, table.cpu(), n)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print("not refused:", i)


@gpu
def test_wrong_contents_are_reported(ops):
    """Page numbers, lengths and starts that only the device sees: nothing is followed out of the buffers, and the
    workspace's error word says so."""
    pool = Pool(ops, 2, 1, 64, 16, [40, 20], "bf16", 8, spare=0)
    q = torch.randn(4, 2, 64).bfloat16().cuda()
    good = ops.flash_paged(q, pool.kv, pool.table, pool.lengths, starts([2, 2]))
    def code(call):
        ws = torch.zeros(ops.paged_attention_workspace(4, 2, 2, 1, 64, 1), dtype=torch.uint8, device="cuda")
        out = call(ws)
        return int(ws[:4].view(torch.int32)), out
    table = pool.table.clone()
    table[0, 1] = pool.k.shape[0]
    got, out = code(lambda ws: ops.flash_paged(q, pool.kv, table, pool.lengths, starts([2, 2]), workspace=ws))
    assert got == 0x601 and torch.equal(out[2:], good[2:])
    got, _ = code(lambda ws: ops.decode_attention_paged(q[:2], pool.kv, table, pool.lengths, workspace=ws))
    assert got == 0x601
    n = torch.tensor([200, 20], dtype=torch.int32).cuda()
    got, out = code(lambda ws: ops.flash_paged(q, pool.kv, pool.table, n, starts([2, 2]), workspace=ws))
    assert got == 0x602 and torch.equal(out[2:], good[2:])
    got, _ = code(lambda ws: ops.decode_attention_paged(q[:2], pool.kv, pool.table, n, workspace=ws))
    assert got == 0x602
    cu = torch.tensor([0, 2, 9], dtype=torch.int32).cuda()
    got, out = code(lambda ws: ops.flash_paged(q, pool.kv, pool.table, pool.lengths, cu, workspace=ws))
    assert got == 0x604


@gpu
def test_empty_calls(ops):
    pool = Pool(ops, 1, 1, 64, 16, [3], "bf16", 9)
    z = torch.zeros(0, 2, 64).bfloat16().cuda()
    zk = torch.zeros(0, 1, 64).bfloat16().cuda()
    none = torch.zeros(0, dtype=torch.int32).cuda()
    assert ops.flash_varlen(z, zk, zk, starts([0])).shape == (0, 2, 64)
    assert ops.flash_paged(z, pool.kv, pool.table, pool.lengths, starts([0])).shape == (0, 2, 64)
    assert ops.decode_attention_paged(z, pool.kv, pool.table[:0], none).shape == (0, 2, 64)
    assert ops.paged_append(zk, zk, pool.kv, pool.table[:0], none) is None


def test_decode_matches_itself_in_any_grouping_sizes():
    """The workspace covers every grouping of a batch, and never shrinks with more of it."""
    lib = L.load()
    size = lib.dab_paged_attention_workspace_size
    assert size(5, 5, 2, 4, 64, 5) >= size(5, 5, 2, 4, 64, 0) > 0
    assert size(600, 5, 2, 4, 64, 0) >= size(5, 5, 2, 4, 64, 0)
    assert size(5, 5, 2, 129, 64, 0) == 0 and size(-1, 5, 2, 4, 64, 0) == 0


# ------------------------------------------------------------------------------------ more edges
@gpu
def test_members_shorter_than_their_prefix(ops):
    """Members that end inside the shared rows, the first one among them; and no member that has all of them."""
    for lens in ([100, 300, 0, 290, 256], [100, 0, 37, 200]):
        pool = Pool(ops, len(lens), 2, 128, 16, lens, "bf16", 21, share=256)
        q = torch.randn(len(lens), 8, 128).bfloat16().cuda()
        cu = torch.tensor([0, len(lens)], dtype=torch.int32).cuda()
        n = torch.tensor([256], dtype=torch.int32).cuda()
        out = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, prefix_cu=cu, prefix_lengths=n)
        for b, m in enumerate(lens):
            k, v = pool.rows(b)
            check(out[b:b + 1], attend64(q[b:b + 1], k, v, [m], 128 ** -0.5), pool.v)


@gpu
@pytest.mark.parametrize("Hq,H,D,dt", [(9, 1, 64, "bf16"), (32, 2, 128, "fp16"), (64, 1, 128, "bf16"), (12, 4, 128, "bf16")])
def test_decode_many_query_heads(ops, Hq, H, D, dt):
    """More than 8 query heads per K / V head take another path than up to 8; with and without a prefix."""
    lens = [700, 513, 40, 1000]
    pool = Pool(ops, 4, H, D, 32, lens, dt, 22, share=512)
    q = (2 * torch.randn(4, Hq, D)).to(DT[dt]).cuda()
    cu = torch.tensor([0, 2, 4], dtype=torch.int32).cuda()
    n = torch.tensor([512, 512], dtype=torch.int32).cuda()
    for kw in ({}, dict(prefix_cu=cu, prefix_lengths=n)):
        out = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, **kw)
        for b, m in enumerate(lens):
            k, v = pool.rows(b)
            check(out[b:b + 1], attend64(q[b:b + 1], k, v, [m], D ** -0.5), pool.v)


@gpu
@pytest.mark.parametrize("D,dt", [(64, "fp16"), (128, "bf16")])
def test_decode_with_rising_scores(ops, D, dt):
    """Scores that grow along the keys move the references of both kinds of pieces, by a little and by a lot."""
    lens = [1500] * 40
    pool = Pool(ops, 40, 1, D, 64, lens, dt, 23, share=640)
    q = torch.ones(40, 4, D).to(DT[dt]).cuda()
    cu = torch.tensor([0, 20], dtype=torch.int32).cuda()
    n = torch.tensor([640], dtype=torch.int32).cuda()
    for step in (0.002, 0.03, -0.03):
        for b in range(40):
            p = torch.arange(1500)
            page, row = pool.table[b].cpu().long()[p // 64].cuda(), (p % 64).cuda()
            pool.k[page, :, row] = (step * p.cuda().float())[:, None, None].to(DT[dt]).expand(-1, 1, D)
        out = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, prefix_cu=cu, prefix_lengths=n)
        for b in (0, 19, 20, 39):
            k, v = pool.rows(b)
            # scores of up to 45 * sqrt(128) = 509 in 32-bit sums: off by 2^-24 * 509 * 8, 2^-12 of a weight; the check's
            # 2^-13 max|v| and the unit roundoffs leave that much room (weights sum to one, values to half of max|v|)
            check(out[b:b + 1], attend64(q[b:b + 1], k, v, [1500], D ** -0.5), pool.v)


@gpu
def test_non_finite_rows_stay_with_those_who_see_them(ops):
    """A NaN in one sequence's own rows, and one in shared rows past a member's length, reach nobody else."""
    lens = [300, 290, 100]
    pool = Pool(ops, 3, 1, 64, 32, lens, "bf16", 24, share=256)
    q = torch.randn(3, 4, 64).bfloat16().cuda()
    cu = torch.tensor([0, 3], dtype=torch.int32).cuda()
    n = torch.tensor([256], dtype=torch.int32).cuda()
    ref = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, prefix_cu=cu, prefix_lengths=n)
    pool.k[pool.table[0, 9].long(), :, 2] = float("nan")  # row 290 of the first
    out = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, prefix_cu=cu, prefix_lengths=n)
    assert out[0].isnan().all() and torch.equal(out[1:], ref[1:])


@gpu
def test_calls_on_streams_and_in_graphs(ops):
    """Calls on two streams at once, and captured ones replayed with new contents of the same tensors, give what
    eager calls give; a captured call leaves its workspace fit for the next."""
    pool = Pool(ops, 6, 2, 128, 16, [900, 40, 700, 0, 333, 512], "bf16", 25, share=0)
    pool2 = Pool(ops, 3, 2, 128, 16, [2000, 100, 1500], "bf16", 26)
    q = torch.randn(6, 8, 128).bfloat16().cuda()
    q2 = torch.randn(300, 8, 128).bfloat16().cuda()
    cu2 = starts([100, 60, 140])
    ref = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths)
    ref2 = ops.flash_paged(q2, pool2.kv, pool2.table, pool2.lengths, cu2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            a = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths)
        with torch.cuda.stream(s2):
            b = ops.flash_paged(q2, pool2.kv, pool2.table, pool2.lengths, cu2)
        got.append((a, b))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, ref) and torch.equal(b, ref2)
    ws = torch.zeros(ops.paged_attention_workspace(300, 6, 8, 2, 128), dtype=torch.uint8, device="cuda")
    out, out2 = torch.empty_like(q), torch.empty_like(q2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s1):
        ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, out=out, workspace=ws)
        ops.flash_paged(q2, pool2.kv, pool2.table, pool2.lengths, cu2, out=out2, workspace=ws)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref) and torch.equal(out2, ref2)
    # other lengths and rows in the same tensors
    pool.lengths.copy_(torch.tensor([33, 900, 0, 128, 500, 1], dtype=torch.int32))
    q.copy_(torch.randn_like(q))
    cu2.copy_(starts([10, 0, 250]))
    want = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths)
    want2 = ops.flash_paged(q2, pool2.kv, pool2.table, pool2.lengths, cu2)
    for _ in range(3):
        out.zero_()
        out2.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2[:260], want2[:260]) and (out2[260:] == 0).all()
    assert int(ws[:4].view(torch.int32)) == 0


@gpu
def test_prompts_cut_and_whole_agree(ops):
    """The same sequences in a small call, whose units are cut into chunks, and in a large one, where they stay whole."""
    g = torch.Generator().manual_seed(27)
    n = [700, 64, 1, 400]
    many = n + [300] * 60
    q, k, v = (torch.randn(sum(many), h, 128, generator=g).bfloat16().cuda() for h in (8, 2, 2))
    big = ops.flash_varlen(q, k, v, starts(many))
    T = sum(n)
    small = ops.flash_varlen(q[:T], k[:T], v[:T], starts(n))
    # each is within one rounding of the output and the weights' 16 bits of the formula
    tol = 2 * (2 * UNIT[torch.bfloat16] + 2.0 ** -13) * v.float().abs().max().item()
    assert (big[:T].float() - small.float()).abs().max().item() <= tol
    at = 0
    for m in n:
        check(small[at:at + m], attend64(q[at:at + m], k[at:at + m], v[at:at + m], torch.arange(1, m + 1), 128 ** -0.5), v)
        at += m


@gpu
def test_long_cache_offsets(ops):
    """Pages whose element offsets pass 2^31: rows there are written and read in place."""
    H, D, ps = 8, 128, 64
    P = (1 << 31) // (H * D * ps) + 40  # about 2^31 elements, 4.3 GB for K and as much for V
    kv = ops.PagedKV.empty(P, H, ps, D, torch.bfloat16, "cuda")
    lens = [150, 97]
    table = torch.tensor([[P - 1, 0, P - 3], [P - 2, P - 9, 1]], dtype=torch.int32).cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(28)
    x, y = (torch.randn(sum(lens), H, D, generator=g).bfloat16().cuda() for _ in range(2))
    ops.paged_append(x, y, kv, table, n, cu_seqlens=starts(lens))
    q = torch.randn(2, 32, D, generator=g).bfloat16().cuda()
    out = ops.decode_attention_paged(q, kv, table, n)
    at = 0
    for b, m in enumerate(lens):
        check(out[b:b + 1], attend64(q[b:b + 1], x[at:at + m], y[at:at + m], [m], D ** -0.5), y)
        at += m
    qq = torch.randn(sum(lens), 8, D, generator=g).bfloat16().cuda()
    assert torch.equal(ops.flash_paged(qq, kv, table, n, starts(lens)), ops.flash_varlen(qq, x, y, starts(lens)))


# ------------------------------------------------------------------------------------ the cache
def test_cache_bookkeeping():
    """Pages, places and groups, on the host alone."""
    from deltaattention_b200.cache import PagedDecodeCache
    c = PagedDecodeCache(2, 6, 4, 2, 64, 12, 16, 64, device="cpu")
    a = c.open(40)
    assert a == 0 and c.lengths.tolist() == [40, 0, 0, 0, 0, 0] and len(c._free) == 9
    c._k[:, c._pages[0][2]] = 3.0
    f = c.fork(a, 4)
    assert f == [1, 2, 3, 4] and len(c._free) == 5  # a page each for the partly filled one
    assert all(c._pages[b][:2] == c._pages[0][:2] for b in f) and len({c._pages[b][2] for b in f}) == 4
    assert all((c._k[:, c._pages[b][2]] == 3).all() for b in f)
    assert c.prefix_cu.tolist() == [0, 1, 5, 5, 5, 5, 5] and c.prefix_lengths.tolist()[:2] == [0, 32]
    assert c.page_table[2, :3].tolist() == c._pages[2]
    c.close(a)
    assert c._users[c._pages[1][0]] == 4 and len(c._free) == 6
    c.close(2)  # the group splits, and the place is anybody's
    assert c._groups == {3: (2, 32)} and c.prefix_cu.tolist()[:3] == [0, 3, 5]
    b = c.open(16)
    assert b == 0
    assert c.open(16) == 2 and c.prefix_cu.tolist()[:3] == [0, 3, 5]
    before = len(c._free)
    c.advance()
    assert c.lengths.tolist() == [17, 41, 17, 41, 41, 0] and len(c._free) == before - 2
    with pytest.raises(RuntimeError, match="free"):
        c.open(64)
    with pytest.raises(RuntimeError, match="consecutive"):
        c.fork(0, 2)
    with pytest.raises(ValueError):
        c.open(65)
    with pytest.raises(ValueError):
        c.close(5)
    for _ in range(7):
        c.advance()
    assert len(c._free) == 3 and c.open(16) == 5
    with pytest.raises(RuntimeError, match="wanted"):
        c.advance()  # 4 sequences are at a page's end, 2 pages are free
    assert c.lengths.tolist() == [24, 48, 24, 48, 48, 16]
    for x in (0, 1, 2, 3, 4, 5):
        c.close(x)
    assert sorted(c._free) == list(range(12)) and not c._groups and c.lengths.sum() == 0
    for bad in (dict(head_dim=32), dict(page_size=8), dict(q_heads=3), dict(num_pages=0)):
        with pytest.raises(ValueError):
            PagedDecodeCache(**{**dict(num_layers=1, places=2, q_heads=4, kv_heads=2, head_dim=64, num_pages=2, page_size=16,
                                       max_length=64, device="cpu"), **bad})


@gpu
@pytest.mark.parametrize("dt,D,ps", [("bf16", 128, 16), ("fp16", 64, 32)])
def test_cache_end_to_end(ops, dt, D, ps):
    """Prompts of different lengths, answers that share one, eager and captured steps, places that close and are taken
    again: every output against the formula over the rows that a plain list of them holds."""
    from deltaattention_b200.cache import PagedDecodeCache
    layers, places, Hq, H, dtype, u = 2, 7, 8, 2, DT[dt], UNIT[DT[dt]]
    g = torch.Generator().manual_seed(30)
    c = PagedDecodeCache(layers, places, Hq, H, D, 80, ps, 300, dtype=dtype, max_tokens=400)
    pos = torch.arange(300).double()[:, None] * 1e4 ** (-torch.arange(0, D, 2).double() / D)
    cos, sin = (torch.cat([f(pos), f(pos)], 1).float().cuda() for f in (torch.cos, torch.sin))
    held = [{} for _ in range(layers)]  # per layer, place -> (rotated K rows, V rows), as rounded in the cache

    def rows(n, h):
        return torch.randn(n, h, D, generator=g).to(dtype)

    def turned(x, p):
        """In 64 bits, rounded to the cache's type (a double's two roundings meet fp32's only at ties)."""
        return rotate64(x.double(), cos.cpu().double()[p], sin.cpu().double()[p]).to(dtype)

    def agree(out, qt, k, v, see):
        # An element whose rotation lies within fp32's error of a tie (2^-22 of it; one in 2^13 to 2^10) may be rounded the
        # other way here: that moves its score by 2 u |q k| / sqrt(D), u / 4 of a weight for |q k| = 1 at D = 64. Two
        # such elements in a row's largest weights: u / 2.
        ref = attend64(qt, k, v, see, D ** -0.5)
        tol = (2 * u + 2.0 ** -13 + 0.5 * u) * v.float().abs().max().item()
        assert (out.cpu().double() - ref).abs().max().item() <= tol

    def prefill(places_, news):
        cu = starts(news)
        for layer in range(layers):
            q, k, v = rows(sum(news), Hq), rows(sum(news), H), rows(sum(news), H)
            out = c.prefill(layer, places_, q.cuda(), k.cuda(), v.cuda(), cu, cos, sin)
            at = 0
            for b, m in zip(places_, news):
                old = c._length[b] - m
                p = torch.arange(old, old + m)
                k0, v0 = held[layer].get(b, (k[:0], v[:0]))
                kk, vv = torch.cat([k0[:old], turned(k[at:at + m], p)]), torch.cat([v0[:old], v[at:at + m]])
                held[layer][b] = kk, vv
                agree(out[at:at + m], turned(q[at:at + m], p), kk, vv, old + torch.arange(1, m + 1))
                at += m

    a, b = c.open(75), c.open(2 * ps)
    prefill([a, b], [75, 2 * ps])
    f = c.fork(a, 3)
    for layer in range(layers):
        for x in f:
            held[layer][x] = held[layer][a]
    q, k, v = (torch.zeros(layers, places, h, D, dtype=dtype, device="cuda") for h in (Hq, H, H))
    out = torch.zeros_like(q)
    graph = None
    for step in range(24):
        if step == 6:
            c.close(f[1])
            d = c.open(50)
            assert d == f[1]  # the middle of the group is taken by another sequence
            prefill([d], [50])
        if step == 9:
            c.close(b)
        c.advance()
        qs, ks, vs = rows(layers * places, Hq), rows(layers * places, H), rows(layers * places, H)
        for t, x in ((q, qs), (k, ks), (v, vs)):
            t.copy_(x.view(t.shape))
        out.fill_(7)
        if step < 3:
            for layer in range(layers):
                c.step(layer, q[layer], k[layer], v[layer], cos, sin, out[layer])
        else:
            if graph is None:
                graph = c.capture_step(q, k, v, out, cos, sin)
            graph.replay()
        for layer in range(layers):
            for x in range(places):
                n = c._length[x]
                if n == 0:
                    assert (out[layer, x] == 0).all()
                    continue
                p = torch.tensor([n - 1])
                i = layer * places + x
                kk, vv = held[layer][x]
                kk, vv = torch.cat([kk[:n - 1], turned(ks[i:i + 1], p)]), torch.cat([vv[:n - 1], vs[i:i + 1]])
                held[layer][x] = kk, vv
                agree(out[layer, x:x + 1], turned(qs[i:i + 1], p), kk, vv, [n])
    assert int(c.err) == 0 and c.workspace_error() == 0


# ------------------------------------------------------------------------- calls at the limits of what is allowed
def test_cache_refuses_wrong_places():
    """Places are host numbers: closed ones, ones outside the batch and ones given twice are refused before anything
    is looked up on the device."""
    from deltaattention_b200.cache import PagedDecodeCache
    c = PagedDecodeCache(1, 3, 4, 2, 64, 8, 16, 64, device="cpu")
    a = c.open(20)
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    for bad in (-1, 1, 3):
        for call in (lambda: c.close(bad), lambda: c.fork(bad, 1), lambda: c.extend(bad, 1),
                     lambda: c.prefill(0, [a, bad], x, x[:, :2], x[:, :2], None)):
            with pytest.raises(ValueError, match="not open"):
                call()
    with pytest.raises(ValueError, match="twice"):
        c.prefill(0, [a, a], x, x[:, :2], x[:, :2], None)
    for bad in (0, -3, 45):
        with pytest.raises(ValueError):
            c.extend(a, bad)
    assert c.lengths.tolist() == [20, 0, 0] and len(c._free) == 6
    c.extend(a, 12)  # fills the second page
    assert c.lengths.tolist() == [32, 0, 0] and len(c._free) == 6
    c.extend(a, 17)
    assert c.lengths.tolist() == [49, 0, 0] and len(c._free) == 4 and c.page_table[0].tolist() == c._pages[0]
    b, d = c.open(48), c.open(16)
    with pytest.raises(RuntimeError, match="wanted"):
        c.extend(b, 16)
    assert c.lengths.tolist() == [49, 48, 16] and (b, d) == (1, 2)
    with pytest.raises(ValueError):
        PagedDecodeCache(1, 3, 258, 2, 64, 8, 16, 64, device="cpu")


@gpu
def test_cache_turns_of_a_conversation(ops):
    """A prompt put in by pieces, and turns of many tokens behind it, one of them of a fork: as one prompt."""
    from deltaattention_b200.cache import PagedDecodeCache
    g = torch.Generator().manual_seed(31)
    c = PagedDecodeCache(1, 4, 8, 2, 64, 64, 16, 400, dtype=torch.float16, max_tokens=200)
    q, k, v = (torch.randn(360, h, 64, generator=g).half().cuda() for h in (8, 2, 2))

    def piece(place, at, n, q=q, k=k, v=v):
        s = slice(at, at + n)
        return c.prefill(0, [place], q[s], k[s], v[s], starts([n]))

    a = c.open(100)
    out = [piece(a, 0, 100)]
    c.extend(a, 137)
    out.append(piece(a, 100, 137))
    b = c.fork(a, 1)[0]
    q2, k2, v2 = (torch.randn(360, h, 64, generator=g).half().cuda() for h in (8, 2, 2))
    c.extend(b, 50)
    turn = piece(b, 237, 50, q2, k2, v2)
    c.extend(a, 123)
    out.append(piece(a, 237, 123))
    check(torch.cat(out), attend64(q, k, v, torch.arange(1, 361), 64 ** -0.5), v)
    kb, vb = (torch.cat([x[:237], y[237:287]]) for x, y in ((k, k2), (v, v2)))
    check(turn, attend64(q2[237:287], kb, vb, torch.arange(238, 288), 64 ** -0.5), vb)
    assert int(c.err) == 0 and c.workspace_error() == 0


@gpu
def test_groups_that_do_not_rise_are_reported(ops):
    """Groups out of order or past the batch: the error word says so, and the step goes on without groups."""
    lens = [300, 290, 100, 280]
    pool = Pool(ops, 4, 2, 64, 32, lens, "bf16", 32, share=256)
    q = torch.randn(4, 8, 64).bfloat16().cuda()
    ref = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths)
    n = torch.tensor([64, 64], dtype=torch.int32).cuda()
    for cu in ([0, 3, 2], [0, 2, 5], [-1, 2, 4], [3, 1, 4], [0, 2 ** 31 - 1, 4]):
        ws = torch.zeros(ops.paged_attention_workspace(4, 4, 8, 2, 64, 2), dtype=torch.uint8, device="cuda")
        out = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, workspace=ws, prefix_lengths=n,
                                         prefix_cu=torch.tensor(cu, dtype=torch.int32).cuda())
        assert int(ws[:4].view(torch.int32)) == 0x604 and torch.equal(out, ref), cu
    for rows in (-5, 2 ** 31 - 1):  # no rows; more than a table holds, and than any member has
        n.fill_(rows)
        pool.table[1:4, :8] = pool.table[0, :8]
        same = torch.tensor([0, 1, 1], dtype=torch.int32).cuda()
        out = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, prefix_cu=same, prefix_lengths=n)
        for b, m in enumerate(lens):
            k, v = pool.rows(b)
            check(out[b:b + 1], attend64(q[b:b + 1], k, v, [m], 64 ** -0.5), pool.v)


@gpu
@pytest.mark.parametrize("B,groups", [(5000, 0), (3000, 700)])
def test_decode_of_thousands_of_sequences(ops, B, groups):
    """More sequences and groups than a block has threads, many of them empty or of one member."""
    g = torch.Generator().manual_seed(B)
    H, D, ps = 1, 64, 16
    lens = torch.randint(0, 90, (B,), generator=g)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), torch.randint(0, B, (groups,), generator=g).sort()[0]]).to(torch.int32)
    table = torch.randint(0, 4000, (B, 6), generator=g)
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        table[a:b, :2] = table[a, :2].clone()
    pages = torch.randn(2, 4000, H, ps, D, generator=g).half()
    q = torch.randn(B, 2, D, generator=g).half()
    kw = dict(prefix_cu=cu.cuda(), prefix_lengths=torch.full((groups,), 32, dtype=torch.int32).cuda()) if groups else {}
    out = ops.decode_attention_paged(q.cuda(), ops.PagedKV(pages[0].cuda(), pages[1].cuda()), table.int().cuda(),
                                     lens.int().cuda(), **kw)
    k, v = (x[table].transpose(1, 2).reshape(B, H, 6 * ps, D).double() for x in pages)
    s = q.double() @ k[:, 0].transpose(1, 2) / 8
    s = s.masked_fill(torch.arange(6 * ps)[None, None] >= lens[:, None, None], -math.inf)
    ref = (s.softmax(-1) @ v[:, 0]).nan_to_num(0.0)
    check(out, ref, v)


@gpu
def test_prompts_by_the_thousand(ops):
    g = torch.Generator().manual_seed(33)
    n = torch.randint(0, 5, (3000,), generator=g).tolist()
    T = sum(n)
    q, k, v = (torch.randn(T, h, 64, generator=g).half() for h in (3, 1, 1))
    out = ops.flash_varlen(q.cuda(), k.cuda(), v.cuda(), starts(n)).cpu()
    own = torch.repeat_interleave(torch.arange(3000), torch.tensor(n))
    ref = torch.empty(T, 3, 64, dtype=torch.float64)
    for a in range(0, T, 500):
        b, lo = min(a + 500, T), max(0, a - 4)
        see = (own[a:b, None] == own[None, lo:b]) & (torch.arange(lo, b)[None] <= torch.arange(a, b)[:, None])
        s = torch.einsum("thd,sd->hts", q[a:b].double(), k[lo:b, 0].double()) / 8
        ref[a:b] = torch.einsum("hts,sd->thd", s.masked_fill(~see, -math.inf).softmax(-1), v[lo:b, 0].double())
    check(out, ref, v)


@gpu
def test_outputs_over_the_queries(ops):
    """``out`` may be q itself: every row is read before it is written, whichever parts a unit is cut into."""
    g = torch.Generator().manual_seed(34)
    lens = [600, 3000, 0, 512, 700] + [513 + i for i in range(60)]
    pool = Pool(ops, len(lens), 2, 128, 16, lens, "bf16", 34, share=512)
    cu = torch.tensor([0, 4, 40], dtype=torch.int32).cuda()
    n = torch.tensor([512, 512], dtype=torch.int32).cuda()
    for Hq in (8, 40):
        q = torch.randn(len(lens), Hq, 128, generator=g).bfloat16().cuda()
        ref = ops.decode_attention_paged(q, pool.kv, pool.table, pool.lengths, prefix_cu=cu, prefix_lengths=n)
        for _ in range(5):
            x = q.clone()
            ops.decode_attention_paged(x, pool.kv, pool.table, pool.lengths, prefix_cu=cu, prefix_lengths=n, out=x)
            assert torch.equal(x, ref)
    for news in ([200, 130, 1], [40] * 150):
        q, k, v = prompt_inputs(news, 8, 2, 128, "bf16")
        ref = ops.flash_varlen(q, k, v, starts(news))
        T = sum(news)
        for _ in range(5):
            x = q.clone()
            ops.flash_varlen(x, k, v, starts(news), out=x)
            assert torch.equal(x[:T], ref[:T]) and torch.equal(x[T:], q[T:])
