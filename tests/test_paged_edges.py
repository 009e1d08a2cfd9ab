"""The paged operators and their cache at the edges of what they take: scratch of one size for calls of many, starts and
positions that only the device sees, calls with nothing in them.

Tolerances are test_paged.py's: 2 u of the largest |v| for 16-bit weights and the output's rounding, 2^-13 of it for
32-bit scores.
"""
import pytest
import torch

from deltaattention_b200 import _lib as L
from test_paged import DT, UNIT, Pool, check, no_device_errors, ops, starts  # noqa: F401  (the fixtures)

gpu = pytest.mark.gpu


def exact(q, k, v, see, scale):
    """test_paged.py's attend64 on the tensors' device, a whole head at a time: q [n, Hq, D], k / v [L, H, D], query i
    sees the first see[i] rows."""
    G = q.shape[1] // k.shape[1]
    hidden = torch.arange(len(k), device=q.device) >= see.to(q.device)[:, None]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for h in range(q.shape[1]):
        s = q[:, h].double() @ k[:, h // G].double().T * scale
        w = torch.where(hidden, 0.0, s.masked_fill(hidden, -torch.inf).softmax(-1))
        out[:, h] = w @ v[:, h // G].double()
    return out.cpu()


# ------------------------------------------------------------------------------------ scratch
@pytest.mark.parametrize("H,G,D", [(8, 4, 128), (1, 1, 64), (4, 7, 128), (128, 1, 64), (2, 128, 64), (300, 1, 64)])
def test_scratch_rises_with_every_size(H, G, D):
    """Scratch for some tokens, sequences and groups serves every call with fewer of them."""
    size = L.load().dab_paged_attention_workspace_size
    for B in (1, 16, 700):
        last = 0
        for T in range(0, 9000 if H > 1 else 90000, 1 if H > 1 else 17):
            now = size(T, B, H, G, D, 0)
            assert now >= last, (T, B)
            last = now
    for T in (1, 500, 2367, 2368, 9000):
        sizes = [size(T, B, H, G, D, 0) for B in range(1, 400)]
        assert sizes == sorted(sizes)
        assert size(T, 50, H, G, D, 20) >= size(T, 50, H, G, D, 3) >= sizes[49]


@gpu
@pytest.mark.parametrize("Hq,H,D,dt,most,news", [
    (32, 8, 128, "bf16", 8192, [1, 300, 2000, 2367, 2368, 3500]), (128, 128, 64, "fp16", 2000, [1, 100, 767, 768, 1030])])
def test_cache_for_long_prompts_takes_short_ones(ops, Hq, H, D, dt, most, news):
    """A cache made for many tokens at a time takes prompts of any fewer, whole and behind others, and steps."""
    from deltaattention_b200.cache import PagedDecodeCache
    g = torch.Generator(device="cuda").manual_seed(40)
    rows = lambda n, h: torch.randn(n, h, D, generator=g, device="cuda").to(DT[dt])  # noqa: E731
    c = PagedDecodeCache(1, 16, Hq, H, D, 80, 128, 5000, dtype=DT[dt], max_tokens=most)
    for n in news:
        a = c.open(n)
        q, k, v = rows(n, Hq), rows(n, H), rows(n, H)
        out = c.prefill(0, [a], q, k, v, starts([n]))
        check(out, exact(q, k, v, torch.arange(1, n + 1), D ** -0.5), v)
        c.extend(a, 37)
        q2, k2, v2 = rows(37, Hq), rows(37, H), rows(37, H)
        out = c.prefill(0, [a], q2, k2, v2, starts([37]))
        k, v = torch.cat([k, k2]), torch.cat([v, v2])
        check(out, exact(q2, k, v, n + torch.arange(1, 38), D ** -0.5), v)
        c.advance()
        x, y, z = rows(16, Hq), rows(16, H), rows(16, H)
        out = c.step(0, x, y, z)
        k, v = torch.cat([k, y[a:a + 1]]), torch.cat([v, z[a:a + 1]])
        check(out[a:a + 1], exact(x[a:a + 1], k, v, torch.tensor([n + 38]), D ** -0.5), v)
        c.close(a)
    assert int(c.err) == 0 and c.workspace_error() == 0


# ------------------------------------------------------------------------- contents that only the device sees
@gpu
@pytest.mark.parametrize("cu", [[0, 512] * 8 + [0], [0, 512, 0, 512], [0, 512, 511], [9, 3, 512], [512, 0]])
@pytest.mark.parametrize("T", [512, 40000])
def test_starts_that_fall(ops, T, cu):
    """Sequences that overlap, over rows that many chunks would be cut from: reported, nothing computed, nothing
    written behind the scratch, and the scratch is fit for the next call. (With 40000 tokens units stay whole.)"""
    B, rows = len(cu) - 1, 128000
    kv = ops.PagedKV(*(torch.randn(1, 1, 256, 64, device="cuda").half() for _ in range(2)))
    table = torch.zeros(B, rows // 256, dtype=torch.int32, device="cuda")
    lengths = torch.full((B,), rows, dtype=torch.int32, device="cuda")
    starts_ = torch.tensor(cu, dtype=torch.int32, device="cuda")
    q = torch.randn(T, 4, 64, device="cuda").half()
    n = ops.paged_attention_workspace(T, B, 4, 1, 64)
    whole = torch.zeros(n + (64 << 20), dtype=torch.uint8, device="cuda")
    ws, guard = whole[:n], whole[n:]
    guard.fill_(77)
    k = torch.randn(T, 1, 64, device="cuda").half()
    for call in (lambda out: ops.flash_paged(q, kv, table, lengths, starts_, out=out, workspace=ws),
                 lambda out: ops.flash_varlen(q, k, k, starts_, out=out, workspace=ws)):
        out = torch.full_like(q, 7.0)
        call(out)
        assert int(ws[:4].view(torch.int32)) == 0x604
        assert (out == 7).all() and (guard == 77).all()
        ws[:4] = 0
        good = starts([100, 200])
        got = ops.flash_varlen(q[:300], k[:300], k[:300], good, workspace=ws)
        for a, b in ((0, 100), (100, 300)):
            check(got[a:b], exact(q[a:b], k[a:b], k[a:b], torch.arange(1, b - a + 1), 64 ** -0.5), k)
        assert int(ws[:4].view(torch.int32)) == 0 and (guard == 77).all()


@gpu
@pytest.mark.parametrize("captured", [False, True])
def test_calls_with_nothing_in_them(ops, captured):
    """A padded call whose tokens belong to no sequence, before and after others on one scratch and one stream."""
    g = torch.Generator(device="cuda").manual_seed(41)
    q = torch.randn(700, 8, 64, generator=g, device="cuda").half()
    k, v = (torch.randn(700, 2, 64, generator=g, device="cuda").half() for _ in range(2))
    cu = starts([300, 0, 390])
    ref = ops.flash_varlen(q, k, v, cu)
    check(ref[:300], exact(q[:300], k[:300], v[:300], torch.arange(1, 301), 64 ** -0.5), v)
    nobody = [torch.zeros(4, dtype=torch.int32, device="cuda"), torch.full((4,), 700, dtype=torch.int32, device="cuda")]
    ws = torch.zeros(ops.paged_attention_workspace(700, 3, 8, 2, 64), dtype=torch.uint8, device="cuda")
    empty, outs = torch.full_like(q, 7.0), [torch.full_like(q, 7.0) for _ in range(40)]

    def calls():
        for i, out in enumerate(outs):
            for _ in range(1 + i % 3):
                ops.flash_varlen(q, k, v, nobody[i % 2], out=empty, workspace=ws)
            ops.flash_varlen(q, k, v, cu, out=out, workspace=ws)

    if captured:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            calls()
        for _ in range(5):
            graph.replay()
    else:
        calls()
    assert (empty == 7).all() and int(ws[:4].view(torch.int32)) == 0
    for out in outs:
        assert torch.equal(out[:690], ref[:690]) and (out[690:] == 7).all()


@gpu
@pytest.mark.parametrize("news,lens,Hq,H,D,dt", [
    ([5, 2], [3, 0], 2, 1, 64, "fp16"), ([300, 40, 200], [170, 40, 333], 8, 2, 128, "bf16"), ([130], [1], 3, 3, 64, "bf16"),
    ([900, 64], [129, 65], 16, 4, 64, "fp16"), ([2500] * 4, [1300] * 4, 32, 8, 64, "bf16")])
def test_queries_before_the_first_row(ops, news, lens, Hq, H, D, dt):
    """More queries than rows: those at negative positions give 0, causal or not, whatever parts the keys are cut into."""
    pool = Pool(ops, len(lens), H, D, 16, lens, dt, 42)
    q = torch.randn(sum(news), Hq, D, generator=torch.Generator().manual_seed(sum(news))).to(DT[dt]).cuda()
    for causal in (True, False):
        out = ops.flash_paged(q, pool.kv, pool.table, pool.lengths, starts(news), causal=causal)
        at = 0
        for b, (m, n) in enumerate(zip(news, lens)):
            k, v = (x.cuda() for x in pool.rows(b))
            none = max(0, m - n)
            assert (out[at:at + none] == 0).all()
            s = slice(at + none, at + m)
            see = n - m + none + torch.arange(1, m - none + 1) if causal else torch.full((m - none,), n)
            if m > none:
                check(out[s], exact(q[s], k, v, see, D ** -0.5), pool.v)
            at += m


@gpu
@pytest.mark.parametrize("news,lens", [([300, 40], [170, 40]), ([2500] * 4, [1300] * 4)])
def test_queries_that_see_nothing_of_rows_that_are_nan(ops, news, lens):
    """A query at a negative position gives 0 whatever the rows hold, in units that are cut and in whole ones."""
    pool = Pool(ops, len(lens), 8, 64, 16, lens, "bf16", 43)
    q = torch.randn(sum(news), 32, 64, generator=torch.Generator().manual_seed(43)).bfloat16().cuda()
    pool.v.fill_(float("nan"))
    for causal in (True, False):
        out = ops.flash_paged(q, pool.kv, pool.table, pool.lengths, starts(news), causal=causal)
        at = 0
        for m, n in zip(news, lens):
            assert (out[at:at + max(0, m - n)] == 0).all() and out[at + max(0, m - n):at + m].isnan().all()
            at += m


# ------------------------------------------------------------------------------------ the cache
@gpu
def test_cache_knows_its_device(ops):
    """The bookkeeping goes to the device that the cache was made on, not to the one current later."""
    from deltaattention_b200.cache import PagedDecodeCache
    c = PagedDecodeCache(1, 2, 2, 1, 64, 4, 16, 64)
    assert c.device == c.page_table.device == c._k.device and c.device.index is not None


@gpu
def test_step_captured_before_anything_else(ops):
    """A caller's own capture of a cache's step, before its first prompt: the prompt's call finds its scratch zeroed
    though the graph has not run yet, and the graph then gives what an eager step gives."""
    from deltaattention_b200.cache import PagedDecodeCache
    g = torch.Generator(device="cuda").manual_seed(45)
    rows = lambda n, h: torch.randn(n, h, 64, generator=g, device="cuda").half()  # noqa: E731
    c = PagedDecodeCache(1, 2, 8, 2, 64, 40, 16, 400, dtype=torch.float16, max_tokens=300)
    ws = c._ws
    assert ws is not None  # made by the capture it would be the graph's, and zeroed by its replays alone
    x, y, z = rows(2, 8), rows(2, 2), rows(2, 2)
    out = torch.zeros_like(x)
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        c.step(0, x, y, z, out=out)
    assert c._ws is ws and int(ws.count_nonzero()) == 0
    a = c.open(300)
    q, k, v = rows(300, 8), rows(300, 2), rows(300, 2)
    got = c.prefill(0, [a], q, k, v, starts([300]))
    check(got, exact(q, k, v, torch.arange(1, 301), 64 ** -0.5), v)
    c.advance()
    graph.replay()
    check(out[a:a + 1], exact(x[a:a + 1], torch.cat([k, y[a:a + 1]]), torch.cat([v, z[a:a + 1]]), torch.tensor([301]), 64 ** -0.5), v)
    assert torch.equal(out, c.step(0, x, y, z)) and int(c.err) == 0 and c.workspace_error() == 0
