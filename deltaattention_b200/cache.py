"""Decode cache with device-resident lengths (native API).

``HybridCompressedCache`` (deltaDecoding.py:111-233, mirrored in ``dropin/deltaDecoding.py``)
keeps the exact-window and total lengths of every layer as Python integers, reads the
largest packed length back from the GPU every 256 tokens (deltaDecoding.py:216-221) and
grows its packed buffers by copying them. ``DeviceDecodeCache`` keeps the same buffers
(shapes, dtypes, layouts) and runs the same kernels, with three differences:

* the ``(exact, total)`` lengths of each layer live in an int64 device tensor, read by the
  update and attention kernels and advanced on the device (by the attention call's last
  kernel in ``step``), so a decode step issues kernel launches only (no host
  synchronisation, no host-side length bookkeeping);
* the packed capacity is fixed at construction (prefill anchors plus the decode steps
  planned: each step appends at most one anchor per head); a full cache sets the update
  kernel's error word (0x201) instead of growing;
* because nothing in a step depends on host values that change per token, a whole
  multi-layer step can be captured once in a CUDA graph and replayed per token
  (``capture_step``).

Outputs and cache contents are bit-identical to the host-length launches of the same
kernels (tests/test_gpu_parity.py).

``Kv4DecodeCache`` keeps the packed history in 4 bits and can go on when it is full: heads are cut
to the entries that drew the most attention.
"""
from __future__ import annotations

import torch

from . import _lib as L
from . import ops


class DeviceDecodeCache:
    """Per-layer hybrid compressed KV cache; lengths on the device."""

    def __init__(self, num_layers, batch, kv_heads, head_dim, capacity, exact_window, dtype=torch.bfloat16,
                 device="cuda", threshold=0.0, use_cosine=False):
        self.num_layers, self.bsz, self.n_kv_heads, self.head_dim = num_layers, batch, kv_heads, head_dim
        self.capacity, self.exact_window_size, self.dtype = int(capacity), int(exact_window), dtype
        self.device = torch.device(device)
        # the reference compares cosine similarity with the raw threshold and Euclidean
        # distance with its square (deltaDecoding.py:75-96)
        self.use_cosine = bool(use_cosine)
        self.threshold = float(threshold) if use_cosine else float(threshold) ** 2
        shp = (num_layers, batch, kv_heads)
        dev = self.device
        self.k_packed = torch.zeros((*shp, self.capacity, head_dim), device=dev, dtype=dtype)
        self.v_packed = torch.zeros_like(self.k_packed)
        self.packed_counts = torch.zeros((*shp, self.capacity), device=dev, dtype=torch.int32)
        self.packed_timestamps = torch.zeros((*shp, self.capacity), device=dev, dtype=torch.int32)
        self.packed_lengths = torch.zeros((num_layers, batch * kv_heads), device=dev, dtype=torch.int32)
        self.k_exact = torch.zeros((*shp, self.exact_window_size, head_dim), device=dev, dtype=dtype)
        self.v_exact = torch.zeros_like(self.k_exact)
        self.seq_state = torch.zeros((num_layers, 2), device=dev, dtype=torch.int64)  # (exact, total) per layer
        self.err = torch.zeros((1,), device=dev, dtype=torch.int32)
        self._ws = None
        self._ws_heads = 0

    def load_prefill(self, layer, k_packed, v_packed, counts, timestamps, k_exact, v_exact, total_len,
                     batch_index=None):
        """The prefill hand-off of ``HybridCompressedCache.initialize_from_prefill``.

        With ``batch_index`` the tensors hold one sequence ([1, Hkv, ...]) and fill that row of
        the batch, so sequences of different lengths (a varlen prefill) are loaded one by one.
        The batch shares the layer's (exact, total) pair, as the reference's cache does; the
        total only stamps the timestamps of anchors appended during decode."""
        p_len = k_packed.shape[2]
        if p_len > self.capacity:
            raise ValueError(f"DeviceDecodeCache: {p_len} packed anchors exceed the capacity {self.capacity}")
        b = slice(None) if batch_index is None else slice(int(batch_index), int(batch_index) + 1)
        self.k_packed[layer, b, :, :p_len] = k_packed
        self.v_packed[layer, b, :, :p_len] = v_packed
        self.packed_counts[layer, b, :, :p_len] = counts
        self.packed_timestamps[layer, b, :, :p_len] = timestamps
        self.packed_lengths[layer].view(self.bsz, self.n_kv_heads)[b] = p_len
        e_len = k_exact.shape[2]
        self.k_exact[layer, b, :, :e_len] = k_exact
        self.v_exact[layer, b, :, :e_len] = v_exact
        self.seq_state[layer, 0] = e_len
        self.seq_state[layer, 1] = int(total_len)

    def _workspace(self, hq):
        if self._ws is None or self._ws_heads != hq:
            lib = L.load()
            nbytes = lib.dab_decode_attention_workspace_size(self.bsz, hq, self.capacity, self.exact_window_size,
                                                             self.head_dim)
            self._ws = torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=self.device)
            self._ws_heads = hq
        return self._ws

    def update(self, layer, k_new, v_new, advance=True):
        """Append one token per (batch, kv-head): k_new / v_new [B, Hkv, 1, d]. Advances the
        layer's lengths on the device (with ``advance=False`` the advance is left to the next
        ``attend(..., advance=True)``)."""
        L.require_cuda(k_new, v_new)
        lib = L.load()
        st = L.stream_of(k_new)
        ke, kp, pc = self.k_exact[layer], self.k_packed[layer], self.packed_counts[layer]
        bd = 16
        while bd < self.head_dim:
            bd <<= 1
        L.check(lib.dab_decode_update_dev(
            L.ptr(k_new), L.ptr(v_new), L.ptr(ke), L.ptr(self.v_exact[layer]), L.ptr(kp),
            L.ptr(self.v_packed[layer]), L.ptr(pc), L.ptr(self.packed_timestamps[layer]),
            L.ptr(self.packed_lengths[layer]), L.ptr(self.seq_state[layer]), self.threshold, self.exact_window_size,
            L.dtype_code(k_new), L.strides(k_new.stride()), L.strides(ke.stride()), L.strides(kp.stride()),
            L.strides(pc.stride()), self.n_kv_heads, self.head_dim, bd, 1 if self.use_cosine else 0,
            self.bsz * self.n_kv_heads, self.capacity, L.ptr(self.err), st), "decode_update_dev")
        if advance:
            L.check(lib.dab_decode_advance(L.ptr(self.seq_state[layer]), 1, st), "decode_advance")

    def attend(self, layer, q, out=None, sm_scale=None, advance=False):
        """Decode attention of q [B, Hq, d] over the layer's packed history and exact window.

        With ``advance`` the call also performs the length advance an ``update(...,
        advance=False)`` left pending: it attends with the advanced window length and steps
        the lengths after its last read."""
        L.require_cuda(q, out)
        B, hq, D = q.shape
        if out is None:
            out = torch.empty_like(q)
        if sm_scale is None:
            sm_scale = D ** -0.5
        lib = L.load()
        st = L.stream_of(q)
        kp, vp, pc = self.k_packed[layer], self.v_packed[layer], self.packed_counts[layer]
        pl = self.packed_lengths[layer].view(self.bsz, self.n_kv_heads)
        ke, ve = self.k_exact[layer], self.v_exact[layer]
        strides = [*q.stride(), *kp.stride(), *vp.stride(), *pc.stride(), *pl.stride(), *ke.stride(), *ve.stride(),
                   *out.stride()]
        ws = self._workspace(hq)
        L.check(lib.dab_decode_attention_dev(
            L.ptr(q), L.ptr(kp), L.ptr(vp), L.ptr(pc), L.ptr(pl), L.ptr(ke), L.ptr(ve), L.ptr(out), L.dtype_code(q),
            L.strides(strides), float(sm_scale), L.ptr(self.seq_state[layer]), 1 if advance else 0,
            self.exact_window_size,
            hq // self.n_kv_heads, B, hq, D, self.capacity, L.ptr(ws), ws.numel(), st), "decode_attention_dev")
        return out

    def step(self, layer, q, k_new, v_new, out=None):
        """One layer's decode step: update, length advance, attention (the reference's order),
        as two launches: the advance rides with the attention call."""
        self.update(layer, k_new, v_new, advance=False)
        return self.attend(layer, q, out, advance=True)

    def lengths(self):
        """(exact, total) per layer, read back to the host (a synchronising call)."""
        return [tuple(int(x) for x in row) for row in self.seq_state.cpu()]

    def capture_step(self, q, k_new, v_new, out):
        """Capture one decode step over every layer in a CUDA graph.

        q / out [layers, B, Hq, d], k_new / v_new [layers, B, Hkv, 1, d] are static device
        buffers: write a token's inputs into them, then ``graph.replay()`` runs the step and
        leaves the result in ``out``. Returns the ``torch.cuda.CUDAGraph``."""
        self._workspace(q.shape[2])
        s = torch.cuda.Stream(self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for layer in range(self.num_layers):
                self.step(layer, q[layer], k_new[layer], v_new[layer], out[layer])
        torch.cuda.current_stream(self.device).wait_stream(s)
        return g


class Kv4DecodeCache:
    """``DeviceDecodeCache`` with the packed history in 4 bits and a way on when it is full.

    An entry of the history takes 172 bytes at head_dim 128 instead of 520 (codes, scales, count,
    timestamp, attention weight; ``ops.kv4_quantize`` gives the format), the exact window stays in
    16 bits. Lengths live on the device as there, so ``step`` and ``evict`` only launch kernels and
    can be captured. Merge and append decisions are those of the 16-bit cache: the last anchor's key
    is kept in 16 bits for the comparison.

    ``packed_lengths`` are [num_layers, B, Hkv], the counts, timestamps and masses [num_layers, B, Hkv, ..]
    (``DeviceDecodeCache`` has its lengths as [num_layers, B * Hkv]).

    Attention adds every entry's weight to ``mass`` (history) and ``exact_mass`` (window; it moves with
    the token into the history). ``evict`` cuts heads to their heaviest entries by it, in place.

    ``err`` (int32 [1] on the device) holds the first error until it is zeroed: 0x201, a token had to be
    appended to a full history and was lost; 0x501, a wait inside an eviction ran out and the cache is
    not valid."""

    def __init__(self, num_layers, batch, kv_heads, head_dim, capacity, exact_window, dtype=torch.bfloat16,
                 device="cuda", threshold=0.0, use_cosine=False, track_mass=True):
        if dtype not in (torch.bfloat16, torch.float16) or head_dim not in (64, 128):
            raise ValueError("Kv4DecodeCache: bf16 / fp16 and head_dim 64 / 128 only")
        if exact_window < 1 or capacity < 1:
            raise ValueError("Kv4DecodeCache: capacity and exact_window must be positive")
        self.num_layers, self.bsz, self.n_kv_heads, self.head_dim = num_layers, batch, kv_heads, head_dim
        self.capacity, self.exact_window_size, self.dtype = int(capacity), int(exact_window), dtype
        self.device = torch.device(device)
        self.threshold, self.similarity = float(threshold), "cosine" if use_cosine else "euclidean"
        shp, dev, cap, W = (num_layers, batch, kv_heads), self.device, self.capacity, self.exact_window_size
        z = lambda *s, dt: torch.zeros((*shp, *s), device=dev, dtype=dt)  # noqa: E731
        self._codes = [z(cap, head_dim // 2, dt=torch.uint8) for _ in range(2)]
        self._scales = [z(cap, head_dim // 16, dt=torch.bfloat16) for _ in range(2)]
        self.packed_counts, self.packed_timestamps = z(cap, dt=torch.int32), z(cap, dt=torch.int32)
        self.packed_lengths = z(dt=torch.int32)
        self.mass = z(cap, dt=torch.float32) if track_mass else None
        self.exact_mass = z(W, dt=torch.float32) if track_mass else None
        self.last_key = z(head_dim, dt=dtype)
        self.k_exact, self.v_exact = z(W, head_dim, dt=dtype), z(W, head_dim, dt=dtype)
        self.seq_state = torch.zeros((num_layers, 2), device=dev, dtype=torch.int64)  # (exact, total) per layer
        # The eviction's workspace begins with its error word, and updates use the same one.
        self._evict_ws = torch.zeros(ops.evict_workspace(batch, kv_heads, cap) if track_mass else 4, device=dev,
                                     dtype=torch.uint8)
        self.err = self._evict_ws[:4].view(torch.int32)
        self.hist = [ops.KV4(self._codes[0][i], self._scales[0][i], self._codes[1][i], self._scales[1][i])
                     for i in range(num_layers)]
        self._ws = {}

    def load_prefill(self, layer, k_packed, v_packed, counts, timestamps, k_exact, v_exact, total_len,
                     batch_index=None, mass=None):
        """``DeviceDecodeCache.load_prefill``, the packed rows going into 4 bits. ``mass`` [B, Hkv, p_len]
        is the weight that the anchors start with (0 by default)."""
        p_len, e_len = k_packed.shape[2], k_exact.shape[2]
        if p_len > self.capacity:
            raise ValueError(f"Kv4DecodeCache: {p_len} packed anchors exceed the capacity {self.capacity}")
        if e_len > self.exact_window_size:
            raise ValueError(f"Kv4DecodeCache: {e_len} exact tokens exceed the window {self.exact_window_size}")
        b = slice(None) if batch_index is None else slice(int(batch_index), int(batch_index) + 1)
        h = self.hist[layer]
        ops.kv4_quantize(k_packed.to(self.dtype), v_packed.to(self.dtype),
                         out=ops.KV4(*(t[b, :, :p_len] for t in (h.k_codes, h.k_scales, h.v_codes, h.v_scales))))
        if p_len:
            self.last_key[layer, b] = k_packed[:, :, p_len - 1]
        self.packed_counts[layer, b, :, :p_len] = counts
        self.packed_timestamps[layer, b, :, :p_len] = timestamps
        self.packed_lengths[layer, b] = p_len
        if self.mass is not None:
            self.mass[layer, b, :, :p_len] = 0.0 if mass is None else mass
            self.exact_mass[layer, b] = 0.0
        self.k_exact[layer, b, :, :e_len] = k_exact
        self.v_exact[layer, b, :, :e_len] = v_exact
        self.seq_state[layer, 0] = e_len
        self.seq_state[layer, 1] = int(total_len)

    def _layer(self, t, layer):
        return None if t is None else t[layer]

    def _workspace(self, name, nbytes):
        """This cache's own scratch. Smaller ones stay for the life of the cache: a captured step may use them."""
        kept = self._ws.setdefault(name, [])
        if not kept or kept[-1].numel() < nbytes:
            kept.append(torch.zeros(nbytes, dtype=torch.uint8, device=self.device))
        return kept[-1]

    def update(self, layer, k_new, v_new, advance=True):
        """Takes one token per (batch, kv-head): k_new / v_new [B, Hkv, 1, d]; ``advance`` as in
        ``DeviceDecodeCache.update``."""
        ops.decode_update_kv4(
            k_new, v_new, self.hist[layer], self.packed_counts[layer], self.packed_timestamps[layer],
            self.packed_lengths[layer], self.last_key[layer], self.k_exact[layer], self.v_exact[layer],
            self.seq_state[layer], threshold=self.threshold, similarity=self.similarity,
            mass=self._layer(self.mass, layer), exact_mass=self._layer(self.exact_mass, layer), err=self.err)
        if advance:
            L.check(L.load().dab_decode_advance(L.ptr(self.seq_state[layer]), 1, L.stream_of(k_new)), "decode_advance")

    def attend(self, layer, q, out=None, sm_scale=None, advance=False):
        """Attention of q [B, Hq, d] over the layer's history and window, adding to their mass."""
        ws = self._workspace("attend", ops.kv4_attention_workspace(
            self.bsz, q.shape[1], self.n_kv_heads, self.head_dim, self.capacity, self.exact_window_size,
            self.mass is not None))
        return ops.decode_attention_kv4(
            q, self.hist[layer], self.packed_counts[layer], self.packed_lengths[layer], self.k_exact[layer],
            self.v_exact[layer], seq_state=self.seq_state[layer], advance=advance, mass=self._layer(self.mass, layer),
            exact_mass=self._layer(self.exact_mass, layer), sm_scale=sm_scale, out=out, workspace=ws)

    def step(self, layer, q, k_new, v_new, out=None):
        """One layer's decode step: update, length advance, attention."""
        self.update(layer, k_new, v_new, advance=False)
        return self.attend(layer, q, out, advance=True)

    def evict(self, layer, budget, trigger=None, keep_first=0, keep_recent=1):
        """Cuts every head of the layer that holds more than ``trigger`` anchors to its ``budget`` heaviest
        (``ops.evict_by_mass``). The last anchor always stays: the next token may merge into it."""
        if self.mass is None:
            raise ValueError("Kv4DecodeCache.evict: the cache does not track attention mass")
        if keep_recent < 1:
            raise ValueError("Kv4DecodeCache.evict: keep_recent must be at least 1")
        h = self.hist[layer]
        ops.evict_by_mass(self.mass[layer], self.packed_lengths[layer],
                          (h.k_codes, h.k_scales, h.v_codes, h.v_scales, self.packed_counts[layer],
                           self.packed_timestamps[layer]), budget, trigger=trigger, keep_first=keep_first,
                          keep_recent=keep_recent, workspace=self._evict_ws)

    def dequantize(self, layer, dtype=None):
        """The history's K and V rows [B, Hkv, capacity, d] (rows past a head's length hold anything)."""
        return ops.kv4_dequantize(self.hist[layer], self.dtype if dtype is None else dtype)

    def lengths(self):
        """(exact, total) per layer, read back to the host (a synchronising call)."""
        return [tuple(int(x) for x in row) for row in self.seq_state.cpu()]

    def capture_step(self, q, k_new, v_new, out, evict=None):
        """``DeviceDecodeCache.capture_step``; with ``evict`` (the arguments of ``evict`` but the layer, as a
        dict) every replay also cuts the heads that have passed the trigger. Run one eager step (and
        eviction) first."""
        s = torch.cuda.Stream(self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for layer in range(self.num_layers):
                self.step(layer, q[layer], k_new[layer], v_new[layer], out[layer])
                if evict is not None:
                    self.evict(layer, **evict)
        torch.cuda.current_stream(self.device).wait_stream(s)
        return g
