"""A decode history in 4 bits: quantisation, update, attention and eviction against plain
implementations in 64 bits.

Tolerances, from the formulas:
* a code is the nearest step, so a value is within half a scale of its element (the scale's bf16
  rounding moves the top of the range by less than half a step), plus fp32's rounding;
* attention: the output is rounded once (its type's unit roundoff, 2^-8 or 2^-11 of it), and a
  weight is off by the error of its score, a 32-bit dot product whose terms sum to at most some
  tens (2^-14 of a weight with room for partial sums sixteen times larger), and by weights held
  in 16 bits and more: 2^-12 of the largest value covers both;
* mass: that share of the added weight, and fp32's rounding of the sum.
Selections, counts, lengths and moved rows are equal.
"""
import ctypes
import math

import pytest
import torch

from deltaattention_b200 import _lib as L

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # unit roundoff: 8 and 11 significant bits
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from deltaattention_b200 import ops as o
    L.load()
    return o


# ------------------------------------------------------------------ plain forms in 64 bits
def values64(codes, scales):
    """The values of code rows, by the documented place of every element."""
    codes, s = codes.cpu(), scales.cpu().double()
    D = codes.shape[-1] * 2
    ng = D // 32
    out = torch.empty((*codes.shape[:-1], D), dtype=torch.float64)
    for d in range(D):
        g, t, i = d // 32, d % 32 // 8, d % 8
        bit = 32 * (t * ng + g) + 4 * i
        c = (codes[..., bit // 8].long() >> (bit % 8)) & 15
        out[..., d] = s[..., ng + g] + s[..., g] * c
    return out


def attend64(q, k, v, counts, lengths, ke, ve, elen, scale):
    """(out, weight added to history, weight added to window), all in 64 bits on the host."""
    q, counts, lengths = q.cpu().double(), counts.cpu(), lengths.cpu()
    B, Hq, D = q.shape
    H, cap, W = counts.shape[1], counts.shape[2], 0 if ke is None else ke.shape[2]
    G = Hq // H
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    wp, we = torch.zeros(B, H, cap, dtype=torch.float64), torch.zeros(B, H, W, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            at = [j for j in range(min(int(lengths[b, h]), cap)) if counts[b, h, j] > 0]
            keys, vals, c = k[b, h, at], v[b, h, at], counts[b, h, at].double()
            if W:
                keys = torch.cat([keys, ke[b, h, :elen].cpu().double()])
                vals = torch.cat([vals, ve[b, h, :elen].cpu().double()])
                c = torch.cat([c, torch.ones(elen, dtype=torch.float64)])
            if not len(keys):
                continue
            z = keys @ q[b, h * G:(h + 1) * G].T * scale + c.log()[:, None]
            w = torch.softmax(z, 0)
            out[b, h * G:(h + 1) * G] = w.T @ vals
            wp[b, h, at] = w[:len(at)].sum(1)
            we[b, h, :elen] = w[len(at):].sum(1)
    return out, wp, we


def evict64(mass, n, budget, first, recent):
    """Indices that a head of n entries keeps, in order."""
    if n <= budget:
        return list(range(n))
    key = [-math.inf if math.isnan(x) else x + 0.0 for x in mass[:n].tolist()]
    nan = [math.isnan(x) for x in mass[:n].tolist()]
    mid = sorted(range(first, n - recent), key=lambda i: (-key[i], nan[i], i))[:budget - first - recent]
    return list(range(first)) + sorted(mid) + list(range(n - recent, n))


# ------------------------------------------------------------------------------ quantisation
@gpu
@pytest.mark.parametrize("B,H,N,D,dt,layout", [
    (1, 1, 1, 64, "bf16", "head"), (2, 3, 17, 128, "fp16", "head"), (1, 8, 777, 128, "bf16", "proj"),
    (3, 2, 100, 64, "fp16", "proj"), (1, 2, 33, 128, "bf16", "columns"), (2, 1, 9, 64, "bf16", "step")])
def test_quantize(ops, B, H, N, D, dt, layout):
    g = torch.Generator().manual_seed(N * D)
    def rows():
        x = torch.randn(B, H, N, D, generator=g) * torch.exp(3 * torch.randn(B, H, N, 1, generator=g)) + 2
        x = x.to(DT[dt]).cuda()
        if layout == "proj":
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "columns":  # the head dim is not the fastest
            return x.transpose(2, 3).contiguous().transpose(2, 3)
        if layout == "step":
            return torch.stack([x, x], -1).flatten(-2)[..., ::2]
        return x
    k, v = rows(), rows()
    hist = ops.kv4_quantize(k, v)
    for x, codes, scales in ((k, hist.k_codes, hist.k_scales), (v, hist.v_codes, hist.v_scales)):
        x = x.cpu().double().unflatten(-1, (D // 32, 32))
        val = values64(codes, scales).unflatten(-1, (D // 32, 32))
        s = scales.cpu().double()
        scale, zero = s[..., :D // 32, None], s[..., D // 32:, None]
        fine = x.isfinite().all(-1)  # a group with an element beyond fp16's range reads back as NaN
        assert val[~fine].isnan().all()
        x, val, scale, zero = x[fine], val[fine], scale[fine], zero[fine]
        lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        assert (zero <= lo).all() and (lo - zero <= 2.0 ** -7 * lo.abs()).all()  # rounded down by at most an ulp
        assert ((scale - (hi - zero) / 15).abs() <= 2.0 ** -8 * scale).all()
        assert ((val - x).abs() <= 0.5 * scale + 2.0 ** -22 * x.abs()).all()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        kd, vd = ops.kv4_dequantize(hist, dtype)
        for y, codes, scales in ((kd, hist.k_codes, hist.k_scales), (vd, hist.v_codes, hist.v_scales)):
            ref = values64(codes, scales).float().to(dtype)
            assert torch.equal(y.cpu().isnan(), ref.isnan()) and torch.equal(y.cpu().nan_to_num(), ref.nan_to_num())


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
def test_quantize_paths_agree(ops, D, dt):
    """Rows in 16-byte pieces (quotients corrected from the reciprocal) and rows at any strides
    (divisions) give the same codes and scales, near ties and far from them."""
    g = torch.Generator().manual_seed(D)
    x = torch.randn(2, 3, 4001, D, generator=g) * torch.exp(2 * torch.randn(2, 3, 4001, 1, generator=g))
    x[0, 0] = torch.randint(-40, 40, (4001, D), generator=g) * 0.25   # quotients on ties
    x[0, 1] = (torch.rand(4001, D, generator=g) < 0.1) * 3.0
    x = x.clamp(-6e4, 6e4).to(DT[dt]).cuda()
    wide = torch.zeros(2, 3, 4001, D + 1, dtype=DT[dt], device="cuda")[..., 1:]
    wide.copy_(x)
    a, b = ops.kv4_quantize(x, -x), ops.kv4_quantize(wide, -wide)
    for u, w in ((a.k_codes, b.k_codes), (a.v_codes, b.v_codes), (a.k_scales, b.k_scales), (a.v_scales, b.v_scales)):
        assert torch.equal(u, w)


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_quantize_special_groups(ops, dt):
    D = 64
    x = torch.zeros(1, 1, 8, D, dtype=DT[dt])
    x[0, 0, 0] = 3.0                                    # constant: scale 0 (or the zero's rounding), value itself
    x[0, 0, 1, :32] = torch.arange(32) / 2.1
    x[0, 0, 1, 5] = float("nan")
    x[0, 0, 2, 40] = float("inf")
    x[0, 0, 3, 40] = -float("inf")
    x[0, 0, 4, :32] = torch.arange(32) % 2 * 6.0e4      # the widest fp16 range
    x[0, 0, 5, :32] = torch.arange(32) * 2.0 ** -24     # fp16's smallest steps
    x[0, 0, 6] = -0.0
    x[0, 0, 7, :32] = -torch.arange(32) - 0.37
    hist = ops.kv4_quantize(x.cuda(), x.cuda())
    k, v = (t.cpu().double()[0, 0] for t in ops.kv4_dequantize(hist, torch.float32))
    assert torch.equal(k.isnan(), v.isnan()) and torch.equal(k[~k.isnan()], v[~v.isnan()])
    ref = x.double()[0, 0]
    bad = torch.zeros(8, D, dtype=torch.bool)
    bad[1, :32] = bad[2, 32:] = bad[3, 32:] = True      # the whole group of a value that is not finite
    assert torch.equal(k.isnan(), bad)
    assert torch.equal(k[0], ref[0]) and torch.equal(k[6], torch.zeros(D, dtype=torch.float64))
    rng = 6.0e4
    assert ((k[4, :32] - ref[4, :32]).abs() <= 0.5 * rng / 15 * (1 + 2.0 ** -8)).all()
    step = 31 * 2.0 ** -24 / 15
    assert ((k[5, :32] - ref[5, :32]).abs() <= 0.5 * step * (1 + 2.0 ** -7)).all()
    assert ((k[7, :32] - ref[7, :32]).abs() <= 0.5 * 31.3 / 15).all()


# ---------------------------------------------------------------------------------- attention
def history(ops, B, H, cap, D, dt, seed, scale_v=1.0):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(B, H, cap, D, generator=g) + torch.randn(1, H, 1, D, generator=g)
    v = torch.randn(B, H, cap, D, generator=g) * scale_v + 0.3
    return ops.kv4_quantize(k.to(DT[dt]).cuda(), v.to(DT[dt]).cuda()), g


def check_attend(out, ref, vmax, dtype):
    err = (out.cpu().double() - ref).abs()
    tol = UNIT[dtype] * ref.abs() + 2.0 ** -12 * vmax
    assert (err <= tol).all(), (err - tol).max().item()


ATTEND = [  # B, Hq, H, D, dtype, capacity, lengths, W, exact_len
    (1, 1, 1, 64, "bf16", 1, [1], 0, 0), (1, 4, 1, 128, "bf16", 5, [0], 3, 1), (1, 2, 2, 128, "fp16", 7, [7, 0], 4, 0),
    (1, 8, 8, 64, "fp16", 513, [1, 15, 16, 17, 31, 33, 512, 513], 100, 100),
    (2, 32, 4, 128, "bf16", 300, [0, 300, 129, 128, 127, 64, 257, 1], 100, 37),
    (1, 12, 4, 128, "bf16", 1000, [999, 1000, 640, 3], 128, 128), (1, 7, 1, 64, "bf16", 130, [130], 1, 1),
    (1, 24, 2, 128, "fp16", 260, [259, 255], 33, 33), (3, 6, 3, 64, "fp16", 64, [64] * 9, 16, 16),
    (1, 4, 2, 128, "bf16", 20000, [20000, 18001], 128, 128), (1, 16, 1, 128, "bf16", 4097, [4097], 512, 500),
]


@gpu
@pytest.mark.parametrize("gaps", [False, True])
@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attention(ops, case, gaps):
    B, Hq, H, D, dt, cap, lens, W, E = case
    dtype = DT[dt]
    hist, g = history(ops, B, H, cap, D, dt, cap + Hq)
    counts = torch.randint(1, 9, (B, H, cap), generator=g).int()
    if gaps:
        drop = torch.rand(B, H, cap, generator=g)
        counts = torch.where(drop < 0.2, torch.where(drop < 0.1, 0, -3), counts).int()
        if cap > 40:
            counts[..., 16:48] = 0  # a whole tile
    lengths = torch.tensor(lens, dtype=torch.int32).view(B, H)
    q = (1.5 * torch.randn(B, Hq, D, generator=g)).to(dtype)
    ke = torch.randn(B, H, W, D, generator=g).to(dtype) if W else None
    ve = torch.randn(B, H, W, D, generator=g).to(dtype) if W else None
    mass, emass = torch.rand(B, H, cap, generator=g), torch.rand(B, H, W, generator=g)
    m, em = mass.cuda(), emass.cuda()
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    args = (dev(q), hist, dev(counts), dev(lengths), dev(ke), dev(ve))
    out = ops.decode_attention_kv4(*args, exact_len=E, mass=m, exact_mass=em)
    plain = ops.decode_attention_kv4(*args, exact_len=E)
    k, v = values64(hist.k_codes, hist.k_scales), values64(hist.v_codes, hist.v_scales)
    ref, wp, we = attend64(q, k, v, counts, lengths, ke, ve, E, D ** -0.5)
    vmax = max(v.abs().max().item(), 0.0 if ve is None else ve.abs().max().item())
    check_attend(out, ref, vmax, dtype)
    check_attend(plain, ref, vmax, dtype)
    for got, was, w in ((m, mass, wp), (em, emass, we)):
        err = (got.cpu().double() - (was.double() + w)).abs()
        assert (err <= 2.0 ** -14 * w + 2.0 ** -23 * got.cpu().abs()).all()
        assert torch.equal(got.cpu()[w == 0], was[w == 0])


SHARED = [  # B, Hq, H, D, dtype, capacity, W: more work than one wave of pieces; more heads than pieces
    (16, 32, 8, 128, "bf16", 1000, 100), (16, 8, 8, 64, "fp16", 1400, 33), (8, 48, 4, 128, "fp16", 3000, 0),
    (8, 20, 4, 64, "bf16", 4700, 64), (60, 60, 30, 128, "bf16", 70, 5), (70, 210, 35, 64, "fp16", 33, 16),
    (9, 8, 8, 64, "bf16", 3000, 16),
]


@gpu
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("case", SHARED, ids=str)
def test_attention_with_many_heads(ops, case, ragged):
    """Pieces that begin and end inside heads, and one piece a head."""
    B, Hq, H, D, dt, cap, W = case
    dtype = DT[dt]
    hist, g = history(ops, B, H, cap, D, dt, cap + Hq)
    counts = torch.randint(1, 9, (B, H, cap), generator=g).int()
    lengths = torch.full((B, H), cap, dtype=torch.int32)
    if ragged:
        counts = torch.where(torch.rand(B, H, cap, generator=g) < 0.1, 0, counts).int()
        lengths = torch.randint(0, cap + 1, (B, H), generator=g).int()
        lengths[torch.rand(B, H, generator=g) < 0.3] = 0
        lengths[1, 0], counts[1, 0] = cap, 0
        lengths[2] = 1
    q = (1.5 * torch.randn(B, Hq, D, generator=g)).to(dtype)
    ke = torch.randn(B, H, W, D, generator=g).to(dtype) if W else None
    ve = torch.randn(B, H, W, D, generator=g).to(dtype) if W else None
    E = W - W // 3
    mass, emass = torch.rand(B, H, cap, generator=g), torch.rand(B, H, W, generator=g)
    m, em = mass.cuda(), emass.cuda()
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    args = (dev(q), hist, dev(counts), dev(lengths), dev(ke), dev(ve))
    out = ops.decode_attention_kv4(*args, exact_len=E, mass=m, exact_mass=em)
    plain = ops.decode_attention_kv4(*args, exact_len=E)
    k, v = values64(hist.k_codes, hist.k_scales), values64(hist.v_codes, hist.v_scales)
    ref, wp, we = attend64(q, k, v, counts, lengths, ke, ve, E, D ** -0.5)
    vmax = max(v.abs().max().item(), 0.0 if ve is None else ve.abs().max().item())
    check_attend(out, ref, vmax, dtype)
    check_attend(plain, ref, vmax, dtype)
    for got, was, w in ((m, mass, wp), (em, emass, we)):
        err = (got.cpu().double() - (was.double() + w)).abs()
        assert (err <= 2.0 ** -14 * w + 2.0 ** -23 * got.cpu().abs()).all()
        assert torch.equal(got.cpu()[w == 0], was[w == 0])


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_attention_masked_places_hold_anything(ops, dt):
    """Entries without tokens, past the length and past exact_len hold NaN and infinities."""
    B, Hq, H, D, cap, W, E = 1, 8, 2, 128, 200, 40, 21
    dtype = DT[dt]
    hist, g = history(ops, B, H, cap, D, dt, 5)
    counts = torch.randint(1, 5, (B, H, cap), generator=g).int()
    lengths = torch.tensor([[150, 77]], dtype=torch.int32)
    counts[0, 0, 3] = counts[0, 0, 60:64] = counts[0, 1, 76] = 0
    q = torch.randn(B, Hq, D, generator=g).to(dtype)
    ke, ve = torch.randn(B, H, W, D, generator=g).to(dtype), torch.randn(B, H, W, D, generator=g).to(dtype)
    k, v = values64(hist.k_codes, hist.k_scales), values64(hist.v_codes, hist.v_scales)
    ref, wp, we = attend64(q, k, v, counts, lengths, ke, ve, E, 0.1)
    for s in (hist.k_scales, hist.v_scales):
        s[0, 0, 3] = float("nan")
        s[0, 0, 60:64] = float("inf")
        s[0, 1, 76] = -float("inf")
        s[0, 0, 150:] = float("nan")
        s[0, 1, 77:] = float("inf")
    ke[:, :, E:], ve[:, :, E:] = float("nan"), float("inf")
    counts[0, 0, 150:] = 4
    m, em = torch.zeros(B, H, cap).cuda(), torch.zeros(B, H, W).cuda()
    out = ops.decode_attention_kv4(q.cuda(), hist, counts.cuda(), lengths.cuda(), ke.cuda(), ve.cuda(), exact_len=E,
                                   sm_scale=0.1, mass=m, exact_mass=em)
    check_attend(out, ref, v[..., :77, :].abs().max().item(), dtype)
    assert ((m.cpu() - wp).abs() <= 2.0 ** -14 * wp + 1e-30).all() and ((em.cpu() - we).abs() <= 2.0 ** -14 * we + 1e-30).all()


@gpu
@pytest.mark.parametrize("G", [2, 6])
@pytest.mark.parametrize("qs,vs", [(2.0 ** -100, 1.0), (0.0, 1.0), (2.0 ** 30, 1.0), (1.0, 2.0 ** 40), (1.0, 2.0 ** -30)])
def test_attention_ranges(ops, G, qs, vs):
    """Queries and values of sizes far from one; the scores' size is put right by sm_scale."""
    B, H, D, cap, W = 1, 2, 128, 777, 20
    g = torch.Generator().manual_seed(31)
    k, v = torch.randn(B, H, cap, D, generator=g), torch.randn(B, H, cap, D, generator=g) * vs
    hist = ops.kv4_quantize(k.bfloat16().cuda(), v.bfloat16().cuda())
    counts, lengths = torch.randint(1, 9, (B, H, cap), generator=g).int(), torch.tensor([[777, 300]], dtype=torch.int32)
    q = (torch.randn(B, G * H, D, generator=g) * qs).bfloat16()
    ke, ve = torch.randn(B, H, W, D, generator=g).bfloat16(), (torch.randn(B, H, W, D, generator=g) * vs).bfloat16()
    scale = D ** -0.5 / (qs if qs > 0 else 1.0)
    out = ops.decode_attention_kv4(q.cuda(), hist, counts.cuda(), lengths.cuda(), ke.cuda(), ve.cuda(), sm_scale=scale)
    vv = values64(hist.v_codes, hist.v_scales)
    ref, _, _ = attend64(q, values64(hist.k_codes, hist.k_scales), vv, counts, lengths, ke, ve, W, scale)
    check_attend(out, ref, max(vv.abs().max().item(), ve.abs().max().item()), torch.bfloat16)


@gpu
def test_attention_extreme_scores(ops):
    """One entry far above the others, after and before them, and scores far below zero."""
    B, H, D, cap = 1, 1, 64, 400
    for at in (0, 17, 399):
        k = torch.zeros(B, H, cap, D)
        k[..., :32] = -torch.arange(32) * 2.0
        k[0, 0, at, :32] = torch.arange(32) * 2.0
        v = torch.randn(B, H, cap, D, generator=torch.Generator().manual_seed(at))
        hist = ops.kv4_quantize(k.bfloat16().cuda(), v.bfloat16().cuda())
        q = torch.ones(B, 2, D).bfloat16()
        q[:, 1] = -1.0
        counts = torch.ones(B, H, cap).int()
        lengths = torch.tensor([[cap]], dtype=torch.int32)
        out = ops.decode_attention_kv4(q.cuda(), hist, counts.cuda(), lengths.cuda())
        vv = values64(hist.v_codes, hist.v_scales)
        ref, _, _ = attend64(q, values64(hist.k_codes, hist.k_scales), vv, counts, lengths, None, None, 0, D ** -0.5)
        check_attend(out, ref, vv.abs().max().item(), torch.bfloat16)


@gpu
def test_attention_views_streams_and_repeats(ops):
    """Views of a larger cache, strided q and out, a side stream, and equal bits when repeated."""
    B, Hq, H, D, cap, W = 2, 8, 2, 128, 333, 48
    dtype = torch.bfloat16
    big = ops.KV4.empty(B, H + 1, cap + 19, D, "cuda")
    for t in (big.k_codes, big.v_codes):
        t.fill_(0x5A)
    for t in (big.k_scales, big.v_scales):
        t.fill_(float("nan"))
    hist = ops.KV4(*(t[:, 1:, 16:16 + cap] for t in (big.k_codes, big.k_scales, big.v_codes, big.v_scales)))
    src, g = history(ops, B, H, cap, D, "bf16", 9)
    for a, b in ((hist.k_codes, src.k_codes), (hist.k_scales, src.k_scales), (hist.v_codes, src.v_codes),
                 (hist.v_scales, src.v_scales)):
        a.copy_(b)
    counts = torch.randint(1, 5, (B, H, cap + 7), generator=g).int().cuda()[..., 5:5 + cap]
    lengths = torch.full((B, H), cap, dtype=torch.int32).cuda()
    q = torch.randn(B, 3, Hq, D, generator=g).to(dtype).cuda()[:, 1]
    out = torch.zeros(B, Hq, 2, D, dtype=dtype).cuda()[:, :, 1]
    ring = torch.randn(B, W, 2 * H, D, generator=g).to(dtype).cuda().transpose(1, 2)
    ke, ve = ring[:, :H], ring[:, H:]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    res = []
    for _ in range(3):
        m, em = torch.zeros(B, H, cap + 7, device="cuda")[..., 5:5 + cap], torch.zeros(B, H, W, device="cuda")
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            ops.decode_attention_kv4(q, hist, counts, lengths, ke, ve, mass=m, exact_mass=em, out=out)
        side.synchronize()
        res.append((out.clone(), m.clone(), em.clone()))
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))
    k, v = values64(hist.k_codes, hist.k_scales), values64(hist.v_codes, hist.v_scales)
    ref, wp, we = attend64(q, k, v, counts, lengths, ke, ve, W, D ** -0.5)
    check_attend(out, ref, max(v.abs().max().item(), ve.abs().max().item()), dtype)
    assert ((res[0][1].cpu() - wp).abs() <= 2.0 ** -14 * wp + 1e-30).all()
    assert ((res[0][2].cpu() - we).abs() <= 2.0 ** -14 * we + 1e-30).all()


@gpu
def test_attention_offsets_past_32_bits(ops):
    """Heads whose rows lie more than 2^32 bytes into the code buffer."""
    D, cap, H = 128, 2 ** 20 + 64, 72  # 64 bytes a row: 4.8e9 bytes
    hist = ops.KV4.empty(1, H, cap, D, "cuda")
    for h in (0, H - 1):
        for t, b in ((hist.k_codes, 0x73), (hist.v_codes, 0x2F)):
            t[0, h, :300].fill_(b)
        for t in (hist.k_scales, hist.v_scales):
            t[0, h, :300] = torch.randn(300, D // 16, generator=torch.Generator().manual_seed(h)).bfloat16().cuda()
    counts = torch.ones(1, H, 300, dtype=torch.int32, device="cuda")
    big = torch.ones(1, 1, cap, dtype=torch.int32, device="cuda").expand(1, H, cap)
    lengths = torch.zeros(1, H, dtype=torch.int32)
    lengths[0, 0] = lengths[0, H - 1] = 300
    q = torch.randn(1, H, D, generator=torch.Generator().manual_seed(1)).bfloat16()
    out = ops.decode_attention_kv4(q.cuda(), hist, big, lengths.cuda())
    part = hist.rows(0, 300)
    k, v = values64(part.k_codes[:, ::H - 1], part.k_scales[:, ::H - 1]), values64(part.v_codes[:, ::H - 1], part.v_scales[:, ::H - 1])
    ref, _, _ = attend64(q[:, ::H - 1], k, v, counts[:, ::H - 1], lengths[:, ::H - 1], None, None, 0, D ** -0.5)
    check_attend(out[:, ::H - 1], ref, v.abs().max().item(), torch.bfloat16)
    assert not out[:, 1:H - 1].any()


# -------------------------------------------------------------------------------------- update
def update_state(ops, B, H, cap, D, W, dt, seed, e):
    hist, g = history(ops, B, H, cap, D, dt, seed)
    dtype = DT[dt]
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    s = dict(hist=hist, k_new=r(B, H, 1, D), v_new=r(B, H, 1, D), k_exact=r(B, H, W, D), v_exact=r(B, H, W, D),
             counts=torch.randint(1, 9, (B, H, cap), generator=g).int().cuda(),
             timestamps=torch.randint(0, 99, (B, H, cap), generator=g).int().cuda(),
             mass=torch.rand(B, H, cap, generator=g).cuda(), exact_mass=torch.rand(B, H, W, generator=g).cuda(),
             lengths=torch.randint(0, cap + 1, (B, H), generator=g).int().cuda(),
             seq_state=torch.tensor([e, 1000 + e]).cuda(), err=torch.zeros(1, dtype=torch.int32).cuda())
    near = torch.where(torch.rand(B, H, 1, generator=g) < 0.5, 0.01, 1.5)
    s["last_key"] = (s["k_exact"][:, :, e % W].cpu().float() + near * torch.randn(B, H, D, generator=g)).to(dtype).cuda()
    return s


@gpu
@pytest.mark.parametrize("B,H,cap,D,W,dt,sim,e", [
    (1, 1, 1, 64, 1, "bf16", "euclidean", 5), (2, 8, 9, 128, 100, "bf16", "euclidean", 137),
    (3, 5, 40, 64, 7, "fp16", "cosine", 7), (16, 8, 3, 128, 5, "fp16", "euclidean", 2 ** 33 + 4),
    (2, 4, 9, 128, 8, "bf16", "cosine", 3)])
def test_update(ops, B, H, cap, D, W, dt, sim, e):
    thr = 0.95 if sim == "cosine" else 0.3 * D ** 0.5
    s = update_state(ops, B, H, cap, D, W, dt, 11 * cap + D, e)
    was = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in s.items()}
    old = ops.KV4(*(t.clone() for t in (s["hist"].k_codes, s["hist"].k_scales, s["hist"].v_codes, s["hist"].v_scales)))
    kw = {k: s[k] for k in ("counts", "timestamps", "lengths", "last_key", "k_exact", "v_exact", "seq_state", "mass",
                            "exact_mass", "err")}
    ops.decode_update_kv4(s["k_new"], s["v_new"], s["hist"], threshold=thr, similarity=sim, **kw)
    slot = e % W
    exp = {k: v.cpu().clone() for k, v in was.items() if torch.is_tensor(v)}
    codes = [t.cpu().clone() for t in (old.k_codes, old.k_scales, old.v_codes, old.v_scales)]
    q1 = ops.kv4_quantize(was["k_exact"][:, :, slot:slot + 1], was["v_exact"][:, :, slot:slot + 1])
    new = [t.cpu() for t in (q1.k_codes, q1.k_scales, q1.v_codes, q1.v_scales)]
    full = merged = added = 0
    for b in range(B):
        for h in range(H):
            if e >= W:
                n = int(exp["lengths"][b, h])
                x, y = was["k_exact"][b, h, slot].cpu().double(), was["last_key"][b, h].cpu().double()
                near = (x @ y / (x.norm() * y.norm()) >= thr) if sim == "cosine" else (x - y).norm() <= thr
                m = was["exact_mass"][b, h, slot].cpu()
                if n > 0 and near:
                    exp["counts"][b, h, n - 1] += 1
                    exp["mass"][b, h, n - 1] += m
                    merged += 1
                elif n < cap:
                    for c, d in zip(codes, new):
                        c[b, h, n] = d[b, h, 0]
                    exp["counts"][b, h, n], exp["timestamps"][b, h, n], exp["mass"][b, h, n] = 1, (1000 + e - W + 2 ** 31) % 2 ** 32 - 2 ** 31, m
                    exp["last_key"][b, h] = was["k_exact"][b, h, slot].cpu()
                    exp["lengths"][b, h] = n + 1
                    added += 1
                else:
                    full += 1
            exp["k_exact"][b, h, slot], exp["v_exact"][b, h, slot] = exp["k_new"][b, h, 0], exp["v_new"][b, h, 0]
            exp["exact_mass"][b, h, slot] = 0
    exp["err"][0] = 0x201 if full else 0
    for name in kw:
        assert torch.equal(s[name].cpu(), exp[name]), name
    for got, want in zip((s["hist"].k_codes, s["hist"].k_scales, s["hist"].v_codes, s["hist"].v_scales), codes):
        assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))
    if B * H > 8 and e >= W:
        assert merged and added


@gpu
@pytest.mark.parametrize("similarity", ["euclidean", "cosine"])
def test_update_decides_as_the_16_bit_cache(ops, similarity):
    """Token by token the same merges, appends and timestamps as DeviceDecodeCache."""
    from deltaattention_b200.cache import DeviceDecodeCache
    B, H, D, W, cap, steps = 2, 4, 64, 6, 64, 60
    thr = 0.97 if similarity == "cosine" else 3.0
    ref = DeviceDecodeCache(1, B, H, D, cap, W, threshold=thr, use_cosine=similarity == "cosine")
    hist = ops.KV4.empty(B, H, cap, D, "cuda")
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    counts, times, lengths, state = z(B, H, cap), z(B, H, cap), z(B, H), torch.zeros(2, dtype=torch.int64, device="cuda")
    ke = torch.zeros(B, H, W, D, dtype=torch.bfloat16, device="cuda")
    ve, last = torch.zeros_like(ke), torch.zeros(B, H, D, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(3)
    x = torch.randn(B, H, 1, D, generator=g)
    for _ in range(steps):
        x = 0.95 * x + 0.31 * torch.randn(B, H, 1, D, generator=g)
        k, v = x.bfloat16().cuda(), torch.randn(B, H, 1, D, generator=g).bfloat16().cuda()
        ref.update(0, k, v)
        ops.decode_update_kv4(k, v, hist, counts, times, lengths, last, ke, ve, state, threshold=thr,
                              similarity=similarity)
        state += 1
    assert torch.equal(lengths.flatten(), ref.packed_lengths[0]) and 0 < lengths.sum() < B * H * (steps - W)
    assert torch.equal(counts, ref.packed_counts[0]) and torch.equal(times, ref.packed_timestamps[0])
    assert torch.equal(ke, ref.k_exact[0]) and torch.equal(ve, ref.v_exact[0])
    k4, _ = ops.kv4_dequantize(hist, torch.float32)
    n = lengths.min().item()
    half = 0.5 * hist.k_scales[:, :, :n, :D // 32].float().repeat_interleave(32, -1)
    assert ((k4[:, :, :n] - ref.k_packed[0][:, :, :n].float()).abs() <= half * (1 + 2.0 ** -20)).all()


# ------------------------------------------------------------------------------------ eviction
EVICT = [  # B, H, cap, lengths, budget, trigger, first, recent, mass
    (1, 1, 2, [2], 1, 1, 0, 0, "equal"), (1, 2, 10, [10, 5], 6, 6, 1, 2, "ties"), (1, 1, 300, [300], 3, 3, 1, 2, "rand"),
    (2, 3, 1000, [1000, 999, 700, 701, 0, 1], 700, 700, 4, 128, "zeros"), (1, 2, 777, [777, 600], 500, 650, 0, 0, "ties"),
    (1, 4, 5000, [5000, 4999, 4097, 2049], 2048, 2048, 16, 33, "rand"), (1, 1, 20001, [20001], 19999, 19999, 0, 1, "rand"),
    (1, 2, 600, [600, 600], 400, 400, 3, 5, "odd"), (1, 1, 40000, [40000], 1, 1, 0, 1, "rand"),
    (1, 2, 4096, [4096, 4096], 1000, 1000, 0, 0, "equal"), (1, 1, 70001, [70000], 35001, 35001, 7, 130, "zeros"),
]


@gpu
@pytest.mark.parametrize("case", EVICT, ids=str)
def test_evict(ops, case):
    B, H, cap, lens, budget, trigger, first, recent, kind = case
    g = torch.Generator().manual_seed(cap + budget)
    mass = torch.exp(4 * torch.randn(B, H, cap, generator=g))
    if kind == "zeros":
        mass = torch.where(torch.rand(B, H, cap, generator=g) < 0.6, 0.0, mass)
    elif kind == "ties":
        mass = torch.randint(0, 4, (B, H, cap), generator=g).float()
    elif kind == "equal":
        mass = torch.full((B, H, cap), 0.25)
    elif kind == "odd":  # what should not be there, in an order of its own
        mass = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-45, -1.0, 2.0])[
            torch.randint(0, 8, (B, H, cap), generator=g)]
    lengths = torch.tensor(lens, dtype=torch.int32).view(B, H)
    hist = ops.KV4.empty(B, H, cap, 64, "cuda")
    rows = [hist.k_codes, hist.k_scales, torch.randn(B, H, cap, 128, generator=g).bfloat16().cuda(),
            torch.arange(cap, dtype=torch.int32).expand(B, H, cap).contiguous().cuda(),
            torch.randn(B, H, cap + 3, 3, generator=g).cuda()[:, :, 1:1 + cap],
            torch.randint(-9, 9, (B, H, cap, 2, 3), generator=g).double().cuda()]
    rows[0].random_(0, 256)
    rows[1].copy_(torch.randn(rows[1].shape, generator=g))
    if not rows[4].is_contiguous():  # entries stay contiguous, heads do not
        assert rows[4].stride(1) == 3 * (cap + 3)
    was = [r.cpu().clone() for r in rows]
    m, n = mass.cuda(), lengths.cuda()
    ops.evict_by_mass(m, n, rows, budget, trigger=trigger, keep_first=first, keep_recent=recent)
    for b in range(B):
        for h in range(H):
            length = int(lengths[b, h])
            if length <= trigger:
                kept = list(range(cap))
                assert int(n[b, h]) == length
            else:
                kept = evict64(mass[b, h], length, budget, first, recent)
                assert len(kept) == budget == int(n[b, h])
                kept = kept + list(range(budget, cap))
            for got, want in zip((m, *rows), (mass, *was)):
                a, w = got[b, h].cpu().contiguous(), want[b, h, kept].contiguous()
                assert torch.equal(a.view(torch.uint8), w.view(torch.uint8))


@gpu
@pytest.mark.parametrize("B,H,cap,budget,first,recent,width", [
    (10, 8, 20000, 9000, 4, 100, 1), (1, 1, 140001, 70000, 3, 64, 2), (1, 2, 900, 611, 0, 7, 1000), (2, 40, 600, 257, 1, 1, 1021)])
def test_evict_long_heads_and_wide_rows(ops, B, H, cap, budget, first, recent, width):
    """Heads longer than one pass of their CTAs holds, and entries of up to 4096 bytes with the mass."""
    g = torch.Generator().manual_seed(cap)
    mass = torch.rand(B, H, cap, generator=g).mul(4096).floor()  # ties too
    n = torch.randint(cap - 300, cap + 1, (B, H), generator=g).int()
    rows = [torch.arange(cap, dtype=torch.int32).expand(B, H, cap).contiguous().cuda(),
            torch.randint(-9, 9, (B, H, cap, width), generator=g).int().cuda()]
    was = [r.cpu().clone() for r in rows]
    m, length = mass.cuda(), n.cuda()
    ops.evict_by_mass(m, length, rows, budget, keep_first=first, keep_recent=recent)
    assert (length == budget).all()
    for b in range(B):
        for h in range(H):
            kept = evict64(mass[b, h], int(n[b, h]), budget, first, recent) + list(range(budget, cap))
            for got, want in zip((m, *rows), (mass, *was)):
                assert torch.equal(got[b, h].cpu(), want[b, h, kept])


@gpu
@pytest.mark.parametrize("kind", ["ends", "ties_before", "ties_between", "thin"])
def test_evict_long_stretches_without_kept_entries(ops, kind):
    """One tile of the result whose entries lie tens of thousands of entries apart."""
    cap, budget = 50000, 900
    g = torch.Generator().manual_seed(len(kind))
    mass = 0.5 * torch.rand(1, 2, cap, generator=g)
    at = torch.tensor([3, 40, 41, 63, 64, 1000, 30011, 30012, 47000])
    mass[..., at] = 2.0
    if kind == "ends":             # the heaviest at both ends
        mass[..., :500] += 1
        mass[..., -391:] += 1
    elif kind == "ties_before":    # more ties at the cut than are kept, near the beginning
        mass[..., 100:2100] = 1.0
    elif kind == "ties_between":   # ties at the cut in the middle of a long stretch
        mass[..., 20000:22000] = 1.0
    else:                          # one entry in some 56
        mass[..., ::56] += 1
    n = torch.tensor([[cap, cap - 7]], dtype=torch.int32)
    rows = [torch.arange(cap, dtype=torch.int32).expand(1, 2, cap).contiguous().cuda(),
            torch.randn(1, 2, cap, 5, generator=g).cuda()]
    was = [r.cpu().clone() for r in rows]
    m, length = mass.cuda(), n.cuda()
    ops.evict_by_mass(m, length, rows, budget, keep_first=1, keep_recent=2)
    assert (length == budget).all()
    for h in range(2):
        kept = evict64(mass[0, h], int(n[0, h]), budget, 1, 2) + list(range(budget, cap))
        for got, want in zip((m, *rows), (mass, *was)):
            assert torch.equal(got[0, h].cpu(), want[0, h, kept])


@gpu
def test_evict_row_limit(ops):
    """Rows of 4096 bytes are the widest."""
    m, n = torch.rand(1, 1, 64, device="cuda"), torch.full((1, 1), 64, dtype=torch.int32, device="cuda")
    row = torch.arange(64 * 1025, dtype=torch.int32, device="cuda").view(1, 1, 64, 1025)
    with pytest.raises((ValueError, RuntimeError)):
        ops.evict_by_mass(m, n, [row], 8)
    assert int(n) == 64
    row = row[..., :1024].contiguous()
    kept = evict64(m[0, 0].cpu(), 64, 8, 0, 0)
    want = row[0, 0, kept].clone()
    ops.evict_by_mass(m, n, [row], 8)
    assert int(n) == 8 and torch.equal(row[0, 0, :8], want)


# ------------------------------------------------------------------------------------ refusals
@gpu
def test_refusals(ops):
    B, H, D, cap, W = 1, 2, 64, 32, 8
    hist, _ = history(ops, B, H, cap, D, "bf16", 1)
    c, n = torch.ones(B, H, cap, dtype=torch.int32, device="cuda"), torch.ones(B, H, dtype=torch.int32, device="cuda")
    q = torch.zeros(B, 4, D, dtype=torch.bfloat16, device="cuda")
    ke = torch.zeros(B, H, W, D, dtype=torch.bfloat16, device="cuda")
    m, em = torch.zeros(B, H, cap, device="cuda"), torch.zeros(B, H, W, device="cuda")
    att = ops.decode_attention_kv4
    x = torch.zeros(B, H, 4, D, dtype=torch.bfloat16, device="cuda")
    bad = [
        lambda: ops.kv4_quantize(x, x[:, :, :3]), lambda: ops.kv4_quantize(x.float(), x.float()),
        lambda: ops.kv4_quantize(x[..., :32], x[..., :32]), lambda: ops.kv4_quantize(x.cpu(), x.cpu()),
        lambda: ops.kv4_quantize(x, x, out=hist), lambda: ops.kv4_dequantize(hist, torch.int32),
        lambda: ops.kv4_dequantize(ops.KV4(hist.k_codes, hist.k_scales, hist.v_codes[:, :, ::2], hist.v_scales)),
        lambda: ops.kv4_dequantize(ops.KV4(hist.k_codes[:, :, ::2], hist.k_scales[:, :, ::2], hist.v_codes[:, :, ::2],
                                           hist.v_scales[:, :, ::2])),
        lambda: ops.kv4_dequantize(ops.KV4(hist.k_codes.int(), hist.k_scales, hist.v_codes, hist.v_scales)),
        lambda: att(q[:, :3], hist, c, n), lambda: att(q.float(), hist, c, n), lambda: att(q, hist, c.long(), n),
        lambda: att(q, hist, c[:, :, 1:], n), lambda: att(q, hist, c, n.flatten()), lambda: att(q, hist, c, n, ke),
        lambda: att(q, hist, c, n, ke, ke, exact_len=W + 1), lambda: att(q, hist, c, n, ke, ke, exact_len=-1),
        lambda: att(q, hist, c, n, ke.half(), ke.half()), lambda: att(q, hist, c, n, ke, ke, advance=True),
        lambda: att(q, hist, c, n, ke, ke, mass=m), lambda: att(q, hist, c, n, ke, ke, mass=m, exact_mass=em[..., 1:]),
        lambda: att(q, hist, c, n, ke, ke, mass=m.double(), exact_mass=em), lambda: att(q, hist, c.cpu(), n),
        lambda: att(q, hist, c, n, out=q.float()), lambda: att(q, hist, c, n, workspace=torch.zeros(8, dtype=torch.uint8, device="cuda")),
        lambda: att(torch.zeros(B, 4, D + 1, dtype=torch.bfloat16, device="cuda")[..., 1:], hist, c, n),
        lambda: ops.evict_by_mass(m, n, [c], 0), lambda: ops.evict_by_mass(m, n, [c], 4, keep_first=3, keep_recent=2),
        lambda: ops.evict_by_mass(m, n, [c], 4, trigger=3), lambda: ops.evict_by_mass(m, n, [c] * 9, 4),
        lambda: ops.evict_by_mass(m, n, [c[:, :, 1:]], 4), lambda: ops.evict_by_mass(m.half(), n, [c], 4),
        lambda: ops.evict_by_mass(m, n, [c.to(torch.uint8)], 4), lambda: ops.evict_by_mass(m, n.long(), [c], 4),
        lambda: ops.evict_by_mass(m, n, [c.cpu()], 4), lambda: ops.evict_by_mass(m, n, [c], 4, keep_first=-1),
        lambda: ops.decode_update_kv4(x[:, :, :2], x[:, :, :2], hist, c, c, n, ke[:, :, 0], ke, ke, n, threshold=1.0),
        lambda: ops.decode_update_kv4(x[:, :, :1], x[:, :, :1], hist, c, c, n, ke[:, :, 0], ke, ke,
                                      torch.zeros(2, dtype=torch.int32, device="cuda"), threshold=1.0),
        lambda: ops.decode_update_kv4(x[:, :, :1], x[:, :, :1], hist, c, c, n, ke[:, :, 0], ke[:, :, :0], ke[:, :, :0],
                                      torch.zeros(2, dtype=torch.int64, device="cuda"), threshold=1.0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()


@gpu
def test_nothing_to_do(ops):
    """No batch, no heads, no rows."""
    for B, H, M in ((0, 2, 4), (2, 0, 4), (2, 2, 0)):
        x = torch.zeros(B, H, M, 64, dtype=torch.bfloat16, device="cuda")
        hist = ops.kv4_quantize(x, x)
        assert ops.kv4_dequantize(hist)[0].shape == x.shape
        c, n = torch.ones(B, H, M, dtype=torch.int32, device="cuda"), torch.zeros(B, H, dtype=torch.int32, device="cuda")
        q = torch.ones(B, 2 * H, 64, dtype=torch.bfloat16, device="cuda")
        assert not ops.decode_attention_kv4(q, hist, c, n).any()
        ops.evict_by_mass(c.float(), n, [c], 3)
    torch.cuda.synchronize()


def test_entries_refuse_on_the_host():
    """The C entries check their arguments before anything is launched."""
    import os
    if not os.path.exists(L.LIB_PATH):
        from deltaattention_b200 import build
        build.build()
    lib = L.load()
    z = (ctypes.c_int64 * 24)()
    p = ctypes.c_void_p(4096)
    said = lambda: lib.dab_last_error().decode()  # noqa: E731
    assert lib.dab_kv4_quantize(None, z, p, z, p, p, z, p, p, z, 2, 1, 1, 1, 64, None) == 1 and "null" in said()
    assert lib.dab_kv4_quantize(p, z, p, z, p, p, z, p, p, z, 0, 1, 1, 1, 64, None) == 1 and "bf16" in said()
    assert lib.dab_kv4_quantize(p, z, p, z, p, p, z, p, p, z, 2, 1, 1, 1, 96, None) == 1 and "head_dim" in said()
    assert lib.dab_kv4_quantize(p, z, p, z, p, p, z, p, p, z, 2, 65536, 1, 1, 64, None) == 1 and "65535" in said()
    odd = ctypes.c_void_p(4104)
    assert lib.dab_kv4_quantize(p, z, p, z, odd, p, z, p, p, z, 2, 1, 1, 1, 64, None) == 1 and "16-byte" in said()
    assert lib.dab_kv4_quantize(p, z, p, z, p, p, z, odd, p, z, 2, 1, 1, 1, 128, None) == 1 and "aligned" in said()
    assert lib.dab_kv4_dequantize(p, p, z, p, p, z, p, p, z, 5, 1, 1, 1, 64, None) == 1 and "dtype" in said()
    att = lambda **k: lib.dab_decode_attention_kv4(  # noqa: E731
        p, p, p, p, p, p, p, k.get("mass"), p, p, p, None, k.get("state"), k.get("adv", 0), k.get("elen", 0), z, 1.0,
        k.get("dt", 2), 1, 1, k.get("G", 4), 64, 16, k.get("W", 8), p, k.get("ws", 1 << 30), None)
    for kw, word in ((dict(ws=1), "workspace"), (dict(G=0), "q-heads"), (dict(elen=9), "exact_len"), (dict(adv=1), "seq_state"),
                     (dict(dt=0), "bf16"), (dict(mass=p), "exact_mass"), (dict(W=-1), "sizes")):
        assert att(**kw) == 1 and word in said(), (kw, said())
    upd = lambda state, D, W: lib.dab_decode_update_kv4(  # noqa: E731
        p, p, p, p, p, p, p, p, None, p, p, p, p, None, state, z, 1.0, 0, 2, 1, 1, D, 16, W, None, None)
    assert upd(None, 64, 8) == 1 and "seq_state" in said()
    assert upd(p, 64, 0) == 1 and "exact_window" in said()
    assert upd(p, 32, 8) == 1 and "head_dim" in said()
    rows, one = (L.P * 1)(4096), (ctypes.c_int64 * 1)(6)
    ev = lambda budget, trigger, first, nrow, ws: lib.dab_evict_by_mass(  # noqa: E731
        p, z, p, z, nrow, rows, one, z, 1, 1, 64, budget, trigger, first, 0, p, ws, None)
    assert ev(0, 4, 0, 0, 4096) == 1 and "budget" in said()
    assert ev(4, 3, 0, 0, 4096) == 1 and "trigger" in said()
    assert ev(4, 4, 5, 0, 4096) == 1 and "keep_first" in said()
    assert ev(4, 4, 0, 9, 4096) == 1 and "row buffers" in said()
    assert ev(4, 4, 0, 1, 4096) == 1 and "multiples of 4" in said()
    assert ev(4, 4, 0, 0, 8) == 1 and "workspace" in said()
    assert lib.dab_evict_by_mass(p, z, p, z, 0, None, None, None, 1, 1, 64, 64, 64, 0, 0, p, 4096, None) == 0  # cannot be longer


# --------------------------------------------------------------------------------- together
def filled_cache(B=2, H=2, D=64, cap=96, W=8, layers=2, dtype=torch.bfloat16, seed=0, **kw):
    from deltaattention_b200.cache import Kv4DecodeCache
    g = torch.Generator().manual_seed(seed)
    c = Kv4DecodeCache(layers, B, H, D, cap, W, dtype=dtype, threshold=3.0, **kw)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    for layer in range(layers):
        n = 60 - 7 * layer
        c.load_prefill(layer, r(B, H, n, D), r(B, H, n, D), torch.randint(1, 5, (B, H, n), generator=g).int().cuda(),
                       torch.arange(0, 4 * n, 4).int().cuda().expand(B, H, n), r(B, H, W, D), r(B, H, W, D), 4 * n)
    return c, g


@gpu
def test_cache_step_against_its_own_state(ops):
    """A step is the update, then attention over the state it leaves, its weights added to the mass."""
    B, H, D, W, Hq = 2, 2, 64, 8, 6
    c, g = filled_cache(B, H, D, W=W)
    for step in range(20):
        q = torch.randn(B, Hq, D, generator=g).bfloat16()
        k, v = torch.randn(B, H, 1, D, generator=g).bfloat16().cuda(), torch.randn(B, H, 1, D, generator=g).bfloat16().cuda()
        for layer in range(2):
            was, ewas = c.mass[layer].clone(), c.exact_mass[layer].clone()
            total, slot = int(c.seq_state[layer, 1]), int(c.seq_state[layer, 0]) % W
            n0 = c.packed_lengths[layer].clone()
            out = c.step(layer, q.cuda(), k, v)
            assert c.lengths()[layer] == (W + step + 1, total + 1)
            h = c.hist[layer]
            kk, vv = values64(h.k_codes, h.k_scales), values64(h.v_codes, h.v_scales)
            ref, wp, we = attend64(q, kk, vv, c.packed_counts[layer], c.packed_lengths[layer], c.k_exact[layer],
                                   c.v_exact[layer], W, D ** -0.5)
            check_attend(out, ref, max(vv.abs().max().item(), c.v_exact[layer].abs().max().item()), torch.bfloat16)
            # the leaving token's mass went to the entry that took it
            n = c.packed_lengths[layer].long()
            assert ((n - n0) <= 1).all()
            was.scatter_add_(2, (n - 1)[..., None], torch.where(n > n0, 0.0, ewas[:, :, slot])[..., None])
            put = torch.where((n > n0)[..., None], ewas[:, :, slot, None], was.gather(2, (n - 1)[..., None]))
            was.scatter_(2, (n - 1)[..., None], put)
            ewas[:, :, slot] = 0
            for got, before, w in ((c.mass[layer], was, wp), (c.exact_mass[layer], ewas, we)):
                err = (got.cpu().double() - (before.cpu().double() + w)).abs()
                assert (err <= 2.0 ** -14 * w + 2.0 ** -23 * got.cpu().abs()).all()
    assert int(c.err) == 0


@gpu
def test_cache_evicts_and_goes_on(ops):
    """Captured steps with eviction run past the capacity and equal the same calls made eagerly."""
    B, H, D, Hq, cap, layers, steps = 2, 2, 64, 4, 72, 2, 90
    cut = dict(budget=40, trigger=70, keep_first=2, keep_recent=5)
    caches = [filled_cache(B, H, D, cap=cap, layers=layers)[0] for _ in range(2)]
    g = torch.Generator().manual_seed(8)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()  # noqa: E731
    q, k, v = r(layers, B, Hq, D), r(layers, B, H, 1, D), r(layers, B, H, 1, D)
    outs = [torch.empty_like(q) for _ in caches]
    for c, o in zip(caches, outs):
        for layer in range(layers):
            c.step(layer, q[layer], k[layer], v[layer], o[layer])
            c.evict(layer, **cut)
    graph = caches[0].capture_step(q, k, v, outs[0], evict=cut)
    fell = 0
    for _ in range(steps):
        for t in (q, k, v):
            t.copy_(r(*t.shape))
        n = caches[0].packed_lengths.clone()
        graph.replay()
        for layer in range(layers):
            caches[1].step(layer, q[layer], k[layer], v[layer], outs[1][layer])
            caches[1].evict(layer, **cut)
        fell += int((caches[0].packed_lengths < n).sum())
        assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[0].float()).all()
    a, b = caches
    assert fell and int(a.err) == 0 and int(a.packed_lengths.max()) <= cut["trigger"]
    for name in ("packed_counts", "packed_timestamps", "packed_lengths", "mass", "exact_mass", "last_key", "k_exact",
                 "seq_state"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    n = a.packed_lengths
    for layer in range(layers):
        for bi in range(B):
            for h in range(H):
                ts = a.packed_timestamps[layer, bi, h, :int(n[layer, bi, h])]
                assert (ts[1:] > ts[:-1]).all() and ts[:2].tolist() == [0, 4]  # in order, the first kept
    assert not L.workspace_errors() or all(c == 0 for c in L.workspace_errors())


@gpu
def test_cache_loads_sequences_one_by_one(ops):
    """batch_index fills one row of the batch; the others keep what they hold."""
    c, g = filled_cache(B=3, layers=1)
    was = [t.clone() for t in (c.hist[0].k_codes, c.hist[0].v_scales, c.packed_counts, c.last_key, c.packed_lengths)]
    k, v = torch.randn(1, 2, 11, 64, generator=g).bfloat16().cuda(), torch.randn(1, 2, 11, 64, generator=g).bfloat16().cuda()
    c.load_prefill(0, k, v, torch.full((1, 2, 11), 3, dtype=torch.int32).cuda(), torch.zeros(1, 2, 11, dtype=torch.int32).cuda(),
                   k[:, :, :8], v[:, :, :8], 99, batch_index=1)
    one = ops.kv4_quantize(k, v)
    assert torch.equal(c.hist[0].k_codes[1:2, :, :11], one.k_codes) and torch.equal(c.hist[0].v_scales[1:2, :, :11], one.v_scales)
    assert torch.equal(c.last_key[0, 1], k[0, :, 10]) and c.packed_lengths[0].tolist() == [[60, 60], [11, 11], [60, 60]]
    now = (c.hist[0].k_codes, c.hist[0].v_scales, c.packed_counts[0], c.last_key[0], c.packed_lengths[0])
    for a, b in zip((was[0], was[1], was[2][0], was[3][0], was[4][0]), now):
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    kd, vd = c.dequantize(0, torch.float32)
    assert torch.equal(kd[1:2, :, :11], ops.kv4_dequantize(one, torch.float32)[0])


@gpu
def test_cache_refusals(ops):
    from deltaattention_b200.cache import Kv4DecodeCache
    c, _ = filled_cache(layers=1)
    x = torch.zeros(2, 2, 97, 64, dtype=torch.bfloat16, device="cuda")
    n = torch.zeros(2, 2, 97, dtype=torch.int32, device="cuda")
    plain = Kv4DecodeCache(1, 1, 1, 64, 8, 4, track_mass=False)
    for call in (lambda: Kv4DecodeCache(1, 1, 1, 96, 8, 4), lambda: Kv4DecodeCache(1, 1, 1, 64, 8, 0),
                 lambda: Kv4DecodeCache(1, 1, 1, 64, 8, 4, dtype=torch.float32),
                 lambda: c.load_prefill(0, x, x, n, n, x[:, :, :8], x[:, :, :8], 1),
                 lambda: c.load_prefill(0, x[:, :, :9], x[:, :, :9], n[:, :, :9], n[:, :, :9], x[:, :, :9], x[:, :, :9], 1),
                 lambda: c.evict(0, 10, keep_recent=0), lambda: c.evict(0, 10, trigger=9), lambda: plain.evict(0, 4)):
        with pytest.raises(ValueError):
            call()
