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
