"""Decoding over a 4-bit history that stays within a budget.

A prompt is prefilled with delta attention, its packed history goes into a ``Kv4DecodeCache``, and
tokens are decoded from one captured CUDA graph whose replays also cut heads that have outgrown
their budget to the entries that drew the most attention. Synthetic layer inputs; prints what the
history takes and how far the 4-bit step is from the 16-bit cache's.

    python examples/decode_kv4.py [--prompt 8192] [--tokens 256] [--layers 2]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from deltaattention_b200 import ops, synth  # noqa: E402
from deltaattention_b200.cache import DeviceDecodeCache, Kv4DecodeCache  # noqa: E402


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompt", type=int, default=8192)
    ap.add_argument("--tokens", type=int, default=256)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args()
    dev, B, Hq, Hkv, D, W, period = torch.device("cuda"), 2, 32, 8, 128, 128, 4
    anchors = -(-a.prompt // period)
    capacity, budget = anchors + 64, anchors // 2
    small = Kv4DecodeCache(a.layers, B, Hkv, D, capacity, W, threshold=3.0, device=dev)
    wide = DeviceDecodeCache(a.layers, B, Hkv, D, anchors + W + a.tokens, W, threshold=3.0, device=dev)
    cos, sin = synth.rope_tables(a.prompt, D, 5e5, torch.bfloat16, dev)
    for layer in range(a.layers):
        q, k, v = synth.layer_inputs(B, Hq, Hkv, a.prompt, D, torch.bfloat16, seed=layer, device=dev)
        _, packed, k_rot = ops.delta_prefill(q, k, v, cos, sin, keep_rate=1 / period, return_packed=True)
        for cache in (small, wide):
            cache.load_prefill(layer, packed.k, packed.v, packed.counts, packed.timestamps, k_rot[:, :, -W:],
                               v[:, :, -W:], a.prompt)

    g = torch.Generator(device=dev).manual_seed(1)
    shape = lambda h, *s: (a.layers, B, h, *s, D)  # noqa: E731
    rand = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)  # noqa: E731
    q, k, v = rand(*shape(Hq)), rand(*shape(Hkv, 1)), rand(*shape(Hkv, 1))
    out, ref = torch.empty_like(q), torch.empty_like(q)
    cut = dict(budget=budget, trigger=capacity - 8, keep_first=4, keep_recent=32)
    for layer in range(a.layers):  # one eager step each, before capture
        small.step(layer, q[layer], k[layer], v[layer], out[layer])
        small.evict(layer, **cut)
        wide.step(layer, q[layer], k[layer], v[layer], ref[layer])
    off = ((out.float() - ref.float()).norm() / ref.float().norm()).item()
    graph = small.capture_step(q, k, v, out, evict=cut)
    longest = 0
    for _ in range(a.tokens - 1):
        for t in (q, k, v):
            t.copy_(rand(*t.shape))
        graph.replay()
        longest = max(longest, int(small.packed_lengths.max()))
    torch.cuda.synchronize()
    entry = lambda n: a.layers * B * Hkv * n  # noqa: E731
    print(f"history: {entry(anchors) * 172 / 2**20:.1f} MiB in 4 bits, {entry(anchors) * 520 / 2**20:.1f} MiB in 16")
    print(f"first step: 4-bit output {off:.3f} off the 16-bit cache's (2-norm, relative)")
    print(f"{a.tokens} tokens: anchors per head at most {longest} (capacity {capacity}, cut to {budget} past "
          f"{cut['trigger']}), error word {int(small.err)}")
    assert int(small.err) == 0 and longest <= capacity


if __name__ == "__main__":
    main()
