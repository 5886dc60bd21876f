"""References in 64 bits and device helpers for the tests of the paged batch."""
from __future__ import annotations

import ctypes as C

import numpy as np

from llmplayer_amd import _lib
from llmplayer_amd import hip_forward_pass as hfp
from llmplayer_amd.paged_batch import PagedKv


def reference_tables(length, grow, free, n_free, blocks, page, max_seq, shared, max_tokens, n_pages):
    """One step, sequence by sequence (llmp_paged_tables)."""
    length, grow = [int(x) for x in length], [int(x) for x in grow]
    n = len(length)
    out = {"blocks": blocks.copy(), "free": free.copy(), "len": np.array(length, np.int32), "n_free": n_free,
           "seq_start": np.zeros(n + 1, np.int32), "positions": np.full(max_tokens, -1, np.int32),
           "slots": np.full(max_tokens, -1, np.int32), "status": 0}
    up = lambda x: -(-x // page)  # noqa: E731
    new = [max(g, 0) for g in grow]
    back = [max(up(a) - shared, 0) if g < 0 else 0 for a, g in zip(length, grow)]
    need = [up(a + x) - up(a) if g >= 0 else 0 for a, x, g in zip(length, new, grow)]
    if n_free < 0 or n_free > n_pages or any(a < 0 or a + x > max_seq for a, x in zip(length, new)) or \
            n_free + sum(back) > n_pages:
        out["status"] = -1
    elif sum(new) > max_tokens:
        out["status"] = -2
    else:
        out["status"] = max(0, sum(need) - n_free - sum(back))
    if out["status"]:
        return out
    stack = [int(x) for x in free[:n_free]]
    for b in range(n):
        if grow[b] < 0:
            stack += [int(x) for x in blocks[b, shared:up(length[b])]]
    out["free"][:len(stack)] = stack
    at = 0
    for b in range(n):
        if grow[b] < 0:
            out["len"][b] = 0
        else:
            for j in range(up(length[b]), up(length[b] + new[b])):
                out["blocks"][b, j] = stack.pop()
            for p in range(length[b], length[b] + new[b]):
                pg = int(out["blocks"][b, p // page])
                out["positions"][at] = p
                out["slots"][at] = pg * page + p % page if 0 <= pg < n_pages else -1
                at += 1
            out["len"][b] = length[b] + new[b]
        out["seq_start"][b + 1] = at
    out["n_free"] = len(stack)
    return out


class Device:
    """Uploads that live as long as this object."""

    def __init__(self):
        self.bufs = []

    def up(self, a) -> int:
        a = np.ascontiguousarray(a)
        b = hfp.DeviceBuffer(max(a.nbytes, 16))
        self.bufs.append(b)
        if a.nbytes:
            b.upload(a)
        return b.ptr

    def down(self, ptr, dtype, shape):
        out = np.empty(shape, dtype)
        _lib.call("llmp_memcpy_dtoh", out.ctypes.data, ptr, out.nbytes, 0)
        return out

    def __enter__(self):
        hfp.init(0)
        return self

    def __exit__(self, *exc):
        for b in self.bufs:
            b.free()


def layer_config(kv: PagedKv, n_heads, layer=0, rope_type=0, rope_sel=_lib.LLMP_ROPE_SEL_NONE, window=0, scale=0.0,
                 softcap=0.0, eps=1e-6, qw=None, kw=None):
    fp = lambda a: None if a is None else a.ctypes.data_as(C.POINTER(C.c_float))  # noqa: E731
    _lib.call("llmp_layer_config", kv.handle, layer, n_heads, kv.n_kv_heads, kv.head_dim, rope_type, rope_sel, window, 0,
              scale, softcap, eps, fp(qw), fp(kw))


def values(planes, w):
    """K or V pages as the fp64 values that they hold."""
    x = planes[w].astype(np.float64)
    if w + "s" in planes:
        x = x * np.repeat(planes[w + "s"].astype(np.float64), 32, -1)
    return x


def reference_attention(planes, blocks, seq_start, positions, q, n_tokens, prefix, page, max_seq, window=0, scale=0.0,
                        softcap=0.0, sinks=None, gate=None):
    """(out, tolerance) fp64 [n_tokens][Hq][D]; NaN rows of out: not to be compared (behind the last
    sequence).

    The tolerance counts the roundings of the split products.  A term q_i k_i of a score is off by at most
    3 * 2^-22 of its magnitude (each operand's two fp16 parts keep 22 bits, the product of the two low
    parts is left out), and by 2^-38 of the largest (the fp16 subnormals below the scaled maximum); the
    D terms' roundings are independent, so a score is off by e = 6 of their standard deviations, the
    fp32 sum's sqrt(D) * 2^-24 included.  The output is then off by max|v| * (2 e + 2^-17): twice e from
    numerator and denominator, the rest from the splits of p and v, exp2 and the joins."""
    K, V = values(planes, "k"), values(planes, "v")
    n_pages, hkv, _, D = K.shape
    hq = q.shape[1]
    scale = scale or 1 / np.sqrt(D)
    out, tol = np.full((n_tokens, hq, D), np.nan), np.zeros((n_tokens, hq, 1))
    for b in range(len(seq_start) - 1):
        for t in range(seq_start[b], seq_start[b + 1]):
            p = int(positions[t])
            out[t] = 0
            if p < 0 or p >= max_seq:
                continue
            j = np.arange(max(0, p + 1 - window) if window else 0, p + 1)
            pages = np.where(j < prefix, blocks[0][j // page], blocks[b][j // page])
            j, pages = j[(pages >= 0) & (pages < n_pages)], pages[(pages >= 0) & (pages < n_pages)]
            if len(j) == 0:
                continue
            k, v = (np.repeat(x[pages, :, j % page], hq // hkv, 1) for x in (K, V))     # [rows][Hq][D]
            s = np.einsum("hd,jhd->hj", q[t].astype(np.float64), k) * scale
            mag = np.sqrt(np.einsum("hd,jhd->hj", q[t].astype(np.float64) ** 2, k ** 2)).max(1) * scale
            big = np.abs(q[t]).max(1) * np.abs(k).max((0, 2)) * scale * D
            err = 6 * mag * (3 * 2.0 ** -22 + np.sqrt(D) * 2.0 ** -24) + big * 2.0 ** -38
            if softcap:
                s = softcap * np.tanh(s / softcap)
                err = err + softcap * 2.0 ** -21
            m = s.max(1)
            if sinks is not None:
                m = np.maximum(m, sinks)
            e = np.exp(s - m[:, None])
            total = e.sum(1) + (np.exp(sinks - m) if sinks is not None else 0)
            out[t] = np.einsum("hj,jhd->hd", e, v) / total[:, None]
            if gate is not None:
                out[t] /= 1 + np.exp(-gate[t].astype(np.float64))
            tol[t] = (np.abs(v).max((0, 2)) * (2 * err + 2.0 ** -17 + np.abs(s).max(1) * 2.0 ** -23))[:, None]
    return out, tol
