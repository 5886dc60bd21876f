"""Host-side mirror of the paged batch (llmp_paged_*): many sequences in one pool of pages, with a
prefix that they share stored and attended once.

The reference serves one conversation per KV cache and reuses a cached prefix by copying its state
(LLMEngine.java:400-421, ConversationCache.java:36-56).  PagedKv is the pool with its tables, and
HipBatchPass the attention section of a forward pass for all of its sequences at once, with
HipForwardPass's configuration and layer semantics."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np

from . import _lib
from ._lib import LlmpError, call
from .hip_forward_pass import DeviceBuffer, LayerSetup, ModelConfig, init


class PagedKv:
    """A paged pool (llmp_paged_create) in memory of its own, and host access to its rows."""

    def __init__(self, n_layers: int, n_pages: int, page_size: int, max_seq: int, n_kv_heads: int, head_dim: int,
                 dtype: int = _lib.LLMP_KV_F32):
        h, nbytes = C.c_uint64(), C.c_uint64()
        call("llmp_paged_create", n_layers, n_pages, page_size, max_seq, n_kv_heads, head_dim, dtype, C.byref(h))
        self.handle = h.value
        self.n_pages, self.page_size, self.max_seq = n_pages, page_size, max_seq
        self.n_kv_heads, self.head_dim, self.dtype = n_kv_heads, head_dim, dtype
        call("llmp_paged_bytes", self.handle, C.byref(nbytes))
        self.nbytes = nbytes.value
        self.pool = DeviceBuffer(self.nbytes)
        call("llmp_paged_bind", self.handle, self.pool.ptr)

    @property
    def is_q8(self) -> bool:
        return self.dtype != _lib.LLMP_KV_F32

    @property
    def width(self) -> int:
        """Blocks of a sequence's table."""
        return -(-self.max_seq // self.page_size)

    def planes(self, layer: int):
        """Device addresses (k, k_scales, v, v_scales) of a layer; scales 0 for fp32."""
        p = [C.c_uint64() for _ in range(4)]
        call("llmp_paged_planes", self.handle, layer, *(C.byref(x) for x in p))
        return tuple(x.value for x in p)

    def _shapes(self):
        s = (self.n_pages, self.n_kv_heads, self.page_size, self.head_dim)
        if not self.is_q8:
            return {"k": (s, np.float32), "v": (s, np.float32)}
        t = s[:3] + (self.head_dim // 32,)
        return {"k": (s, np.int8), "ks": (t, np.float32), "v": (s, np.int8), "vs": (t, np.float32)}

    def read(self, layer: int, stream: int = 0) -> dict:
        """A layer's planes: k and v [page][head][row][dim] fp32, or int8 with the scales ks and vs."""
        k, ks, v, vs = self.planes(layer)
        at, out = {"k": k, "ks": ks, "v": v, "vs": vs}, {}
        for w, (shape, dt) in self._shapes().items():
            out[w] = np.empty(shape, dt)
            call("llmp_memcpy_dtoh", out[w].ctypes.data, at[w], out[w].nbytes, stream)
        return out

    def write(self, layer: int, planes: dict, stream: int = 0) -> None:
        """The inverse of read."""
        k, ks, v, vs = self.planes(layer)
        at = {"k": k, "ks": ks, "v": v, "vs": vs}
        for w, (shape, dt) in self._shapes().items():
            a = np.ascontiguousarray(planes[w], dt).reshape(shape)
            call("llmp_memcpy_htod", at[w], a.ctypes.data, a.nbytes, stream)

    def destroy(self) -> None:
        if self.handle:
            call("llmp_kv_destroy", self.handle)
            self.handle = 0
        self.pool.free()


class HipBatchPass(LayerSetup):
    """The attention section (HipForwardPass) for up to max_seqs sequences in one paged pool.

    The first prefix_len positions of every sequence are one prefix: its pages are held once, in
    everyone's table, and read once per layer-call.  prefixStep and forwardBatch compute it, part by
    part.  After that a step is step() (the tables of all sequences, on the GPU, from the lengths and
    setGrow), then per layer forwardBatch on device projections; nothing in it needs a length on the
    host, so it can be captured.  Sequences are rows of fixed place: one whose grow is negative has
    ended and gives its own pages back; setLengths begins its row again behind the prefix."""

    def __init__(self, config: ModelConfig, max_seq_len: int, n_pages: int, page_size: int, max_seqs: int,
                 max_tokens: int, prefix_len: int = 0,
                 qk_norm: Optional[Sequence[Optional[tuple]]] = None, device: int = 0,
                 kv_dtype: int = _lib.LLMP_KV_F32, sinks: Optional[Sequence[Optional[np.ndarray]]] = None):
        c = config
        if c.use_layer_norm or c.head_count % c.head_count_kv:
            raise LlmpError("HipBatchPass", 6, "configuration not supported by the HIP attention path")
        if prefix_len % page_size:
            raise ValueError(f"prefix of {prefix_len} rows: whole pages of {page_size} are shared")
        init(device)
        self.config, self.max_seq_len, self.prefix_len = c, max_seq_len, prefix_len
        self.max_seqs, self.max_tokens = max_seqs, max_tokens
        self.kv = PagedKv(c.block_count, n_pages, page_size, max_seq_len, c.head_count_kv, c.head_size, kv_dtype)
        self._upload_rope()
        for layer in range(c.block_count):
            self.configure_layer(layer, qk_norm[layer] if qk_norm is not None else None)
            if sinks is not None and sinks[layer] is not None:
                self.set_sinks(layer, sinks[layer])
        self.shared_blocks = prefix_len // page_size
        self._shared_now = prefix_len
        if self.shared_blocks > n_pages:
            raise ValueError("the prefix has more pages than the pool")
        i4 = lambda n: DeviceBuffer(4 * n)  # noqa: E731
        self.gpuLen, self.gpuGrow = i4(max_seqs), i4(max_seqs)
        self.gpuFree, self.gpuNFree, self.gpuStatus = i4(n_pages), i4(1), i4(1)
        self.gpuBlocks = i4(max_seqs * self.kv.width)
        self.gpuSeqStart = i4(max_seqs + 1)
        self.gpuPositions, self.gpuSlots = i4(max_tokens), i4(max_tokens)
        self.gpuQ, self.gpuXb2 = i4(max_tokens * c.q_dim), i4(max_tokens * c.q_dim)
        blocks = np.full((max_seqs, self.kv.width), -1, np.int32)
        blocks[:, :self.shared_blocks] = np.arange(self.shared_blocks)
        self.gpuBlocks.upload(blocks)
        free = np.full(n_pages, -1, np.int32)
        free[:n_pages - self.shared_blocks] = np.arange(n_pages - 1, self.shared_blocks - 1, -1)
        self.gpuFree.upload(free)
        self.gpuNFree.upload(np.array([n_pages - self.shared_blocks], np.int32))
        self.setLengths(np.zeros(max_seqs, np.int32))

    def setLengths(self, lengths: np.ndarray) -> None:
        """Rows that each sequence has.  A row that begins anew behind the prefix has prefix_len."""
        self.gpuLen.upload(np.ascontiguousarray(lengths, np.int32).reshape(self.max_seqs))

    def lengths(self) -> np.ndarray:
        return self.gpuLen.download(np.int32)

    def setGrow(self, grow: np.ndarray) -> None:
        self.gpuGrow.upload(np.ascontiguousarray(grow, np.int32).reshape(self.max_seqs))

    def prefixStep(self, start: int, n_tokens: int) -> None:
        """The next forwardBatch calls take prefix tokens [start, start + n_tokens)."""
        if start < 0 or n_tokens < 1 or n_tokens > self.max_tokens or start + n_tokens > self.prefix_len:
            raise ValueError(f"prefix tokens [{start}, {start + n_tokens}) of {self.prefix_len}")
        at = np.full(self.max_tokens, -1, np.int32)
        at[:n_tokens] = np.arange(start, start + n_tokens)   # pages 0, 1, ... in order: slot = position
        self.gpuPositions.upload(at)
        self.gpuSlots.upload(at)
        self.gpuSeqStart.upload(np.concatenate([[0], np.full(self.max_seqs, n_tokens)]).astype(np.int32))
        self._shared_now = 0

    def step(self, stream: int = 0) -> None:
        """Tables of one step from the lengths and grow (setGrow); the lengths advance in place."""
        self._shared_now = self.prefix_len
        call("llmp_paged_tables", self.kv.handle, self.max_seqs, self.shared_blocks, self.max_tokens,
             self.gpuLen.ptr, self.gpuGrow.ptr, self.gpuFree.ptr, self.gpuNFree.ptr, self.gpuBlocks.ptr,
             self.gpuLen.ptr, self.gpuNFree.ptr, self.gpuSeqStart.ptr, self.gpuPositions.ptr,
             self.gpuSlots.ptr, self.gpuStatus.ptr, stream)

    def status(self) -> int:
        """0, or why the last step did nothing (llmp_paged_tables)."""
        return int(self.gpuStatus.download(np.int32)[0])

    def forwardBatch(self, layerIdx: int, q: int, k: int, v: int, in_type: int = _lib.LLMP_IN_F32,
                     max_len: int = 0, gate: int = 0, stream: int = 0) -> None:
        """One layer's attention of the step's tokens from the device projections q, k, v (addresses of
        [max_tokens] rows, fp32 or bf16) into gpuXb2."""
        c = self.config
        call("llmp_paged_append", self.kv.handle, layerIdx, self.max_tokens, self.gpuPositions.ptr,
             self.gpuSlots.ptr, in_type, q, c.q_dim, k, c.kv_dim, v, c.kv_dim, self.gpuQ.ptr, c.q_dim, stream)
        call("llmp_paged_attn", self.kv.handle, layerIdx, self.max_seqs, self.max_tokens, self._shared_now, max_len,
             self.gpuSeqStart.ptr, self.gpuPositions.ptr, self.gpuBlocks.ptr, self.gpuQ.ptr, c.q_dim, gate,
             self.gpuXb2.ptr, c.q_dim, stream)

    def downloadOut(self) -> np.ndarray:
        return self.gpuXb2.download(np.float32).reshape(self.max_tokens, self.config.q_dim)

    def sync(self, stream: int = 0) -> None:
        call("llmp_stream_sync", stream)

    def close(self) -> None:
        for name in ("gpuLen", "gpuGrow", "gpuFree", "gpuNFree", "gpuStatus", "gpuBlocks", "gpuSeqStart",
                     "gpuPositions", "gpuSlots", "gpuQ", "gpuXb2"):
            b = getattr(self, name, None)
            if b is not None:
                b.free()
        if getattr(self, "kv", None) is not None:
            self.kv.destroy()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()
