"""The operators of the 4-bit decode history at the edges of what they take: long flat sums, short heads in
large capacities, values near the ends of their types, workspaces, limits and refusals."""
import pytest
import torch

from deltaattention_b200 import _lib as L
from test_kv4 import DT, UNIT, ops  # noqa: F401  (ops: the fixture)

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------- long flat histories
def device_rows64(codes, scales):
    """(codes, scale of every element, zero of every element) of code rows, by the documented place of every
    element, in 64 bits on their device."""
    D = codes.shape[-1] * 2
    ng = D // 32
    c = torch.empty((*codes.shape[:-1], D), dtype=torch.float64, device=codes.device)
    for d in range(D):
        bit = 32 * (d % 32 // 8 * ng + d // 32) + 4 * (d % 8)
        c[..., d] = (codes[..., bit // 8] >> (bit % 8) & 15).double()
    s = scales.double().repeat_interleave(32, -1)
    return c, s[..., :D], s[..., D:]


@gpu
@pytest.mark.parametrize("D,G,dt", [(64, 1, "fp16"), (128, 4, "bf16"), (128, 4, "fp16"), (64, 6, "bf16"), (128, 8, "fp16")])
def test_attention_of_long_flat_histories(ops, D, G, dt):
    """Nearly equal weights over 100003 entries of values around zero: the output is some hundred times smaller
    than the sums of p scale code and of p zero that make it up.

    The bound: the output's rounding, and 2^-21 of the sum of the terms' sizes. A matrix product of 16 entries
    rounds its sum in the 23rd bit or so; 4 of them at most (two parts of the weights, 32 entries) may add up
    before the zeros are taken into the sum. Weights in 16 bits are off at random, and 10^5 of them
    average to less than 2^-24."""
    H, n = 64, 100003
    g = torch.Generator(device="cuda").manual_seed(D + G)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=DT[dt])  # noqa: E731
    hist = ops.kv4_quantize(rand(1, H, n, D), rand(1, H, n, D))
    q = 0.05 * rand(1, H * G, D)
    ones = torch.ones(1, 1, n, dtype=torch.int32, device="cuda").expand(1, H, n)
    out = ops.decode_attention_kv4(q, hist, ones, torch.full((1, H), n, dtype=torch.int32, device="cuda"))
    for h in range(H):
        c, s, z = device_rows64(hist.k_codes[0, h], hist.k_scales[0, h])
        w = torch.softmax((c * s + z) @ q[0, h * G:(h + 1) * G].double().T * D ** -0.5, 0)
        c, s, z = device_rows64(hist.v_codes[0, h], hist.v_scales[0, h])
        ref, terms = w.T @ (c * s + z), w.T @ (c * s + z.abs())
        err = (out[0, h * G:(h + 1) * G].double() - ref).abs()
        tol = UNIT[DT[dt]] * ref.abs() + 2.0 ** -25 + 2.0 ** -21 * terms
        assert (err <= tol).all(), (h, (err / terms).max().item())


# ------------------------------------------------------- eviction of short heads in large capacities
def kept64(mass, n, budget, first, recent):
    """Indices that a head of n > budget entries keeps, in order: a stable sort of the weights in 64 bits."""
    mid = torch.sort(mass[first:n - recent].double(), descending=True, stable=True).indices[:budget - first - recent]
    return torch.cat([torch.arange(first), first + mid.sort().values, torch.arange(n - recent, n)])


@gpu
@pytest.mark.parametrize("B,H,cap,budget,first,recent,lens", [
    (1, 8, 5000, 20, 2, 3, (21, 31, 32, 33, 64, 100, 255, 256)),         # 2 CTAs a head
    (1, 8, 8448, 100, 0, 1, (101, 250, 120, 128, 129, 256, 257, 3)),     # 4
    (2, 4, 20000, 512, 4, 32, (700, 513, 512, 800, 1024, 1025, 2047, 20000)),  # 8
    (1, 2, 131072, 256, 0, 0, (257, 300)), (1, 1, 140001, 1, 0, 1, (2,)), (1, 1, 40000, 33, 1, 1, (34,)),
    (2, 4, 32768, 256, 16, 100, (257, 511, 513, 769, 1023, 1793, 2049, 300))])
def test_evict_short_heads_in_large_capacities(ops, B, H, cap, budget, first, recent, lens):
    """Capacities that give a head several CTAs, and heads with fewer tiles than CTAs."""
    g = torch.Generator().manual_seed(cap + budget)
    lengths = torch.tensor(lens, dtype=torch.int32).view(B, H)
    mass = torch.randint(0, 50, (B, H, cap), generator=g).float()  # ties too
    for rows in ([torch.arange(cap, dtype=torch.int32).expand(B, H, cap).contiguous()],
                 [torch.arange(cap, dtype=torch.int32).expand(B, H, cap).contiguous(),
                  torch.randint(-9, 9, (B, H, cap, 40), generator=g).int()]):
        m, n, moved = mass.cuda(), lengths.cuda(), [r.cuda() for r in rows]
        ops.evict_by_mass(m, n, moved, budget, keep_first=first, keep_recent=recent)
        assert torch.equal(n.cpu(), lengths.clamp(max=budget))
        for b in range(B):
            for h in range(H):
                length, kept = int(lengths[b, h]), torch.arange(cap)
                if length > budget:
                    kept[:budget] = kept64(mass[b, h], length, budget, first, recent)
                for got, want in zip((m, *moved), (mass, *rows)):
                    assert torch.equal(got[b, h].cpu(), want[b, h, kept])


@gpu
def test_evict_from_two_threads(ops):
    """Host threads whose rows want different amounts of shared memory do not refuse one another's calls."""
    import threading
    cap, budget, rounds = 200, 70, 400
    errors, heads = [], []

    def work(width, seed):
        try:
            g = torch.Generator().manual_seed(seed)
            mass, rows = torch.rand(1, 2, cap, generator=g), torch.randint(-9, 9, (1, 2, cap, width), generator=g).int()
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                m0, r0, n = mass.cuda(), rows.cuda(), torch.empty(1, 2, dtype=torch.int32, device="cuda")
                for _ in range(rounds):
                    m, r = m0.clone(), r0.clone()
                    ops.evict_by_mass(m, n.fill_(cap), [r], budget)
            stream.synchronize()
            heads.append((mass, rows, r.cpu(), n.cpu()))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in ((1000, 1), (60, 2), (500, 3))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for mass, rows, r, n in heads:
        assert (n == budget).all()
        for h in range(2):
            assert torch.equal(r[0, h, :budget], rows[0, h, kept64(mass[0, h], cap, budget, 0, 0)])


# --------------------------------------------------------------------------------- the cache
def small_cache(layers=2, B=2, H=2, D=64, cap=96, W=8, n=50, seed=0, **kw):
    from deltaattention_b200.cache import Kv4DecodeCache
    g = torch.Generator().manual_seed(seed)
    c = Kv4DecodeCache(layers, B, H, D, cap, W, threshold=3.0, **kw)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()  # noqa: E731
    for layer in range(layers):
        c.load_prefill(layer, r(B, H, n, D), r(B, H, n, D), torch.randint(1, 5, (B, H, n), generator=g).int().cuda(),
                       torch.arange(n).int().cuda().expand(B, H, n), r(B, H, W, D), r(B, H, W, D), 4 * n)
    return c, r


@gpu
def test_cache_reports_evictions_error_word(ops, monkeypatch):
    """What an eviction writes into the first word of its workspace is seen in ``err``, and stays there."""
    c, r = small_cache()
    given, evict = [], ops.evict_by_mass

    def noting(*a, workspace=None, **kw):
        given.append(workspace)
        return evict(*a, workspace=workspace, **kw)

    monkeypatch.setattr(ops, "evict_by_mass", noting)
    c.evict(0, 30)
    c.evict(1, 30)
    assert int(c.err) == 0 and (c.packed_lengths == 30).all()
    for ws in list(given):
        ws[:4].view(torch.int32).fill_(0x501)  # as a wait that ran out does
        assert int(c.err) == 0x501
        c.evict(0, 20)
        assert int(c.err) == 0x501
        c.err.zero_()
    full, r = small_cache(cap=50)
    for layer in range(2):
        full.update(layer, 9 * r(2, 2, 1, 64), r(2, 2, 1, 64))
    assert int(full.err) == 0x201
    off, _ = small_cache(track_mass=False)
    assert off.err.shape == c.err.shape == (1,) and off.err.dtype == c.err.dtype == torch.int32 and int(off.err) == 0
    codes = L.workspace_errors()
    assert not any(codes), codes


def test_cache_keeps_scratch_of_captured_steps():
    """A buffer that was handed out lives as long as the cache, also when a later call needs a larger one."""
    import weakref

    from deltaattention_b200.cache import Kv4DecodeCache
    c = Kv4DecodeCache.__new__(Kv4DecodeCache)
    c._ws, c.device = {}, torch.device("cpu")
    first = weakref.ref(c._workspace("attend", 100))
    assert c._workspace("attend", 60) is first()
    larger = c._workspace("attend", 200)
    assert larger.numel() >= 200 and first() is not None and first().data_ptr() != larger.data_ptr()
    assert c._workspace("attend", 200) is larger and c._workspace("attend", 100).numel() >= 100


@gpu
def test_captured_step_after_calls_with_more_heads(ops):
    """A captured step does not write where later tensors are."""
    (c, r), (eager, _) = small_cache(layers=1), small_cache(layers=1)
    q, k, v = r(1, 2, 4, 64), r(1, 2, 2, 1, 64), r(1, 2, 2, 1, 64)
    outs = torch.empty_like(q), torch.empty_like(q)
    for cache, out in zip((c, eager), outs):
        cache.step(0, q[0], k[0], v[0], out[0])
    size = ops.kv4_attention_workspace(2, 4, 2, 64, 96, 8)
    graph = c.capture_step(q, k, v, outs[0])
    wide = r(2, 64, 64)
    for cache in (c, eager):
        cache.attend(0, wide)
    others = [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(64)]
    for _ in range(3):
        graph.replay()
        eager.step(0, q[0], k[0], v[0], outs[1][0])
    assert all((t == 0x5A).all() for t in others)
    assert torch.equal(*outs) and torch.equal(c.mass, eager.mass)


# ----------------------------------------------------------------- quantisation by the formula
FIFTEENTH = torch.tensor(1 / 15, dtype=torch.float32)


def plain_quantize(x, half=False):
    """(codes, scales, zeros) of rows [.., D] by the formula, one fp32 operation at a time; with ``half`` of half the
    elements, the scales and zeros doubled (the same numbers, without fp32's limit on the range)."""
    x = x.float().cpu().unflatten(-1, (-1, 32)) * (0.5 if half else 1.0)
    i = x.amin(-1).view(torch.int32)
    zero = ((i + (i < 0).int() * 0xFFFF) & -0x10000).view(torch.float32)
    scale = ((x.amax(-1) - zero) * FIFTEENTH).bfloat16().float()
    code = ((x - zero[..., None]) / scale[..., None]).round().clamp(0, 15)
    code = torch.where(scale[..., None] == 0, 0.0, code)
    return code.flatten(-2), scale * (2 if half else 1), zero * (2 if half else 1)


def check_quantized(ops, x, half=False):
    """Both paths of the hand-off and the token update against the formula."""
    B, H, N, D = x.shape
    codes, scale, zero = plain_quantize(x, half)
    wide = torch.zeros(B, H, N, D + 1, dtype=x.dtype, device="cuda")[..., 1:]
    wide.copy_(x)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    taken = ops.KV4.empty(B, H, N, D, "cuda")
    lengths, state = z(B, H), torch.tensor([1, 1], device="cuda")
    last, new = torch.zeros(B, H, D, dtype=x.dtype, device="cuda"), torch.zeros(B, H, 1, D, dtype=x.dtype, device="cuda")
    for n in range(N):  # every row leaves a window of one and is appended
        ops.decode_update_kv4(new, new, taken, z(B, H, N), z(B, H, N), lengths, last, x[:, :, n:n + 1].clone(),
                              x[:, :, n:n + 1].clone(), state, threshold=2.0, similarity="cosine")
        assert (lengths == n + 1).all()
    for hist in (ops.kv4_quantize(x, x), ops.kv4_quantize(wide, wide), taken):
        for c, s in ((hist.k_codes, hist.k_scales), (hist.v_codes, hist.v_scales)):
            assert torch.equal(s.cpu().float(), torch.cat([scale, zero], -1))
            assert torch.equal(device_rows64(c, s)[0].cpu().float(), codes)


@gpu
@pytest.mark.parametrize("dt,low", [("bf16", 5), ("fp16", 2)])
def test_quantize_scales_between_two_numbers(ops, dt, low):
    """Ranges of 15 (m + 1/2) steps of bf16: the fifteenth lies between two bf16 numbers, and the format's product
    with the fp32 number next to 1/15 decides, not a division's rounding to even."""
    g = torch.Generator().manual_seed(15)
    r = 15 * torch.arange(257, 512, 2)            # 15 times an odd number of 9 bits
    b = (r >> low << low) if low == 2 else torch.where(r < 4096, r >> 4 << 4, r >> 5 << 5)
    x = torch.rand(len(r), 64, generator=g) * r[:, None] - (r - b)[:, None]
    x = torch.minimum(torch.maximum(x, (b - r)[:, None].float()), b[:, None].float()).to(DT[dt])
    x[:, 3], x[:, 40], x[:, 20], x[:, 63] = (b - r).to(DT[dt]), (b - r).to(DT[dt]), b.to(DT[dt]), b.to(DT[dt])
    x = torch.cat([x, x * 2.0 ** -9, x * 2.0 ** 2, -x]).view(2, 2, len(r), 64)
    _, scale, zero = plain_quantize(x)
    divided = ((x.float().unflatten(-1, (2, 32)).amax(-1) - zero) / 15).bfloat16().float()
    assert 0.2 < (divided != scale).float().mean() < 0.8  # the ranges are as meant
    check_quantized(ops, x.cuda())


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_quantize_tiny_groups(ops, D):
    """bf16 groups down to the smallest subnormals, where a scale may round to a third of what it should be, or to 0,
    and has no reciprocal in fp32."""
    g = torch.Generator().manual_seed(D)
    x = torch.randn(2, 3, 120, D, generator=g)
    x[0, 0] += 3 * torch.randn(120, 1, generator=g)
    x[0, 1, :, :D // 2] = (torch.rand(120, D // 2, generator=g) < 0.1).float()
    x = (x * 2.0 ** (-92 - torch.arange(120) % 48)[:, None].double()).bfloat16()
    check_quantized(ops, x.cuda())


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_quantize_ranges_past_fp32(ops, D):
    """Finite bf16 groups whose range is above the largest fp32 number."""
    g = torch.Generator().manual_seed(D)
    top = torch.finfo(torch.bfloat16).max
    x = (torch.rand(2, 2, 70, D, generator=g) * 2 - 1).mul(top).bfloat16()
    x[..., 0], x[..., 31], x[..., 32], x[..., D - 1] = -top, top, -0.75 * top, 0.5 * top
    x[1, :, :, 5] = 0.0
    assert x.isfinite().all()
    check_quantized(ops, x.cuda(), half=True)
    k, v = ops.kv4_dequantize(ops.kv4_quantize(x.cuda(), x.cuda()), torch.float32)
    _, scale, _ = plain_quantize(x, half=True)
    step = scale.repeat_interleave(32, -1)
    for y in (k, v):
        assert y.isfinite().all() and ((y.cpu().double() - x.double()).abs() <= 0.501 * step.double()).all()


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_read_back_at_the_types_limits(ops, dt):
    """Groups that reach a type's largest numbers read back finite, half a step or a rounding away at most."""
    g = torch.Generator().manual_seed(1)
    top = torch.finfo(DT[dt]).max
    x = ((torch.rand(1, 2, 200, 64, generator=g, dtype=torch.float64) * 2 - 1) * top).to(DT[dt])
    x[0, 0, :, ::7], x[0, 0, :, 1::7] = top, -top
    x[0, 1] = (0.9 + 0.1 * torch.rand(200, 64, generator=g, dtype=torch.float64)).mul(top).to(DT[dt])
    x[0, 1, ::2] *= -1
    x[0, 1, :, 5::32] = x[0, 1, :, 5:6].sign() * top
    assert x.isfinite().all()
    hist = ops.kv4_quantize(x.cuda(), x.cuda())
    step = hist.k_scales[..., :2].cpu().double().repeat_interleave(32, -1)
    for out in (torch.float32, DT[dt]):
        for y in ops.kv4_dequantize(hist, out):
            y = y.cpu().double()
            near = 0.501 * step + UNIT.get(out, 2.0 ** -24) * y.abs() + (2.0 ** -7 * top if dt == "fp16" else 0.0)
            assert y.isfinite().all() and ((y - x.double()).abs() <= near).all()  # fp16's zeros round down to bf16
    x[0, :, ::3, 40] = float("inf")
    x[0, :, 1::3, 41] = float("nan")
    x[0, :, 2::3, 42] = -float("inf")
    for y in ops.kv4_dequantize(ops.kv4_quantize(x.cuda(), x.cuda()), DT[dt]):
        assert y[..., 32:].isnan().all() and y[..., :32].isfinite().all()


# ------------------------------------------------------------------------- workspaces and limits
@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(L.LIB_PATH):
        from deltaattention_b200 import build
        build.build()
    return L.load()


def test_workspace_alignment_is_checked_on_the_host(lib):
    import ctypes
    z, p = (ctypes.c_int64 * 24)(), ctypes.c_void_p(4096)
    said = lambda: lib.dab_last_error().decode()  # noqa: E731
    for odd in (1, 4, 8):
        ws = ctypes.c_void_p(8192 + odd)
        assert lib.dab_decode_attention_kv4(p, p, p, p, p, p, p, None, p, p, p, None, None, 0, 0, z, 1.0, 2, 1, 1, 4, 64, 16,
                                            8, ws, 1 << 30, None) == 1 and "workspace must be 16-byte aligned" in said()
        assert lib.dab_evict_by_mass(p, z, p, z, 0, None, None, None, 1, 1, 64, 4, 4, 0, 0, ws, 1 << 30, None) == 1
        assert "workspace must be 16-byte aligned" in said()


@gpu
def test_workspaces_that_are_refused(ops):
    B, H, D, cap = 1, 2, 64, 32
    x = torch.zeros(B, H, cap, D, dtype=torch.bfloat16, device="cuda")
    hist, q = ops.kv4_quantize(x, x), torch.zeros(B, 4, D, dtype=torch.bfloat16, device="cuda")
    c, n = torch.ones(B, H, cap, dtype=torch.int32, device="cuda"), torch.full((B, H), cap, dtype=torch.int32, device="cuda")
    m = torch.zeros(B, H, cap, device="cuda")
    room = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    for ws in (room[8:], room[1:], room[::2], room[:1].expand(1 << 16), room.view(torch.float32)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.decode_attention_kv4(q, hist, c, n, workspace=ws)
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.evict_by_mass(m, n, [c], 4, workspace=ws)
    ops.decode_attention_kv4(q, hist, c, n, workspace=room[16:])
    ops.evict_by_mass(m, n, [c], 4, workspace=room.zero_()[16:])
    assert (n == 4).all() and not room.view(torch.int32)[4]


def test_attention_sizes_past_its_indexes_are_refused(lib):
    """Columns of a row of scores, and the units of work of one kv-head, are 32-bit numbers."""
    import ctypes
    z, p = (ctypes.c_int64 * 24)(), ctypes.c_void_p(4096)
    said = lambda: lib.dab_last_error().decode()  # noqa: E731
    most = 2 ** 30 - 1
    for G, cap, W in ((4, most, most), (1024, 64, 2 ** 28), (1024, 2 ** 29, 0)):
        assert lib.dab_decode_attention_kv4(p, p, p, p, p, p, p, p, p, p, p, p, None, 0, 0, z, 1.0, 2, 1, 1, G, 64, cap, W, p,
                                            (1 << 64) - 1, None) == 1 and "too long" in said(), (G, cap, W, said())


@gpu
def test_expanded_tensors_are_not_written(ops):
    """Heads or sequences that share memory may be read; written they would spoil one another."""
    B, H, D, cap, W = 2, 3, 64, 32, 4
    x = torch.randn(B, H, cap, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    hist = ops.kv4_quantize(x, x)
    z = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731

    def forms(make, *size):  # expanded over batch, over heads, over both
        for s in ((1, H), (B, 1), (1, 1)):
            yield make(*s, *size).expand(B, H, *size)

    f32, bf = (lambda *s: z(*s, dt=torch.float32)), (lambda *s: z(*s, dt=torch.bfloat16))
    q, n = x[:, :, 0].repeat_interleave(2, 1), torch.full((B, H), cap, dtype=torch.int32, device="cuda")
    c, m, em, ring = z(B, H, cap) + 1, f32(B, H, cap), f32(B, H, W), bf(B, H, W, D)
    bad = []
    for t in forms(f32, cap):
        bad += [lambda t=t: ops.evict_by_mass(t, n, [c], 4),
                lambda t=t: ops.decode_attention_kv4(q, hist, z(1, 1, cap).expand_as(t), n, mass=t, exact_mass=None)]
    for t in forms(z):
        bad.append(lambda t=t: ops.evict_by_mass(m, t, [c], 4))
    for t in forms(z, cap):
        bad.append(lambda t=t: ops.evict_by_mass(m, n, [c, t], 4))
    for t in forms(f32, W):
        bad.append(lambda t=t: ops.decode_attention_kv4(q, hist, c, n, ring, ring, mass=m, exact_mass=t))
    for t in (bf(1, 2 * H, D).expand(B, 2 * H, D), bf(B, 1, D).expand(B, 2 * H, D)):
        bad.append(lambda t=t: ops.decode_attention_kv4(q, hist, c, n, out=t))
    wide = ops.KV4.empty(1, H, cap, D, "cuda")
    shared = ops.KV4(*(t.expand(B, *t.shape[1:]) for t in (wide.k_codes, wide.k_scales, wide.v_codes, wide.v_scales)))
    bad.append(lambda: ops.kv4_quantize(x, x, out=shared))
    new, state = x[:, :, :1], torch.tensor([5, 9], device="cuda")

    def update(**kw):
        a = dict(hist=hist, counts=c, timestamps=z(B, H, cap), lengths=z(B, H), last_key=bf(B, H, D), k_exact=ring,
                 v_exact=ring.clone(), seq_state=state, threshold=1.0, mass=m, exact_mass=em)
        ops.decode_update_kv4(new, new, **{**a, **kw})

    bad.append(lambda: update(hist=shared))
    for t, u in zip(forms(z, cap), forms(f32, cap)):
        bad.append(lambda t=t, u=u: update(counts=t, timestamps=t, mass=u))
    for t in forms(z):
        bad.append(lambda t=t: update(lengths=t))
    for t in forms(bf, D):
        bad.append(lambda t=t: update(last_key=t))
    for t in (*forms(bf, W, D), bf(B, H, 1, D).expand(B, H, W, D)):
        bad.append(lambda t=t: update(k_exact=t, v_exact=t))
    for t in forms(f32, W):
        bad.append(lambda t=t: update(exact_mass=t))
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    assert (n == cap).all()
    # read, they are taken: one sequence's history for all of them, counts and window of one head for all
    one = ops.KV4(*(t[:1].expand_as(t) for t in (hist.k_codes, hist.k_scales, hist.v_codes, hist.v_scales)))
    ones, w = (z(1, 1, cap) + 1).expand(B, H, cap), x[:1, :1, :W].expand(B, H, W, D)
    out = ops.decode_attention_kv4(q, one, ones, n[:1, :1].expand(B, H), w, w)
    same = ops.KV4(*(t.contiguous() for t in (one.k_codes, one.k_scales, one.v_codes, one.v_scales)))
    assert torch.equal(out, ops.decode_attention_kv4(q, same, c, n, w.contiguous(), w.contiguous()))
    update()
    one_by_one = torch.zeros(1, 1, cap, device="cuda").expand(1, 1, cap)  # a stride of a single head is no stride
    ops.evict_by_mass(one_by_one, n[:1, :1], [], 4)
    assert n.flatten().tolist() == [4] + [cap] * 5


def test_lengths_that_share_memory_are_refused(lib):
    """A head's CTAs read its length one after another, and the first writes it: it has to be the head's own."""
    import ctypes
    z, p = (ctypes.c_int64 * 24)(), ctypes.c_void_p(4096)
    for B, H, st, fine in ((2, 1, (0, 7), False), (1, 2, (7, 0), False), (2, 3, (1, 1), False), (2, 3, (2, 1), False),
                           (4, 3, (2, 3), False), (2, 3, (-2, 1), False), (2, 3, (3, 1), True), (2, 3, (1, 2), True),
                           (2, 3, (2, 3), True), (1, 1, (0, 0), True), (5, 1, (1, 0), True)):
        ls = (ctypes.c_int64 * 2)(*st)
        rc = lib.dab_evict_by_mass(p, z, p, ls, 0, None, None, None, B, H, 64, 4, 4, 0, 0, p, 8, None)
        said = lib.dab_last_error().decode()
        assert rc == 1 and ("workspace too small" if fine else "share memory") in said, (B, H, st, said)


@gpu
def test_queries_without_heads_to_read(ops):
    """q-heads over a history of no heads are refused like any other number that does not fit."""
    x = torch.zeros(1, 0, 4, 64, dtype=torch.bfloat16, device="cuda")
    c, n = torch.zeros(1, 0, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, 0, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ops.decode_attention_kv4(torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda"), ops.kv4_quantize(x, x), c, n)
