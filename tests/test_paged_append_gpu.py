"""GPU checks of llmp_paged_append: queries against the rotation in 64 bits, stored rows bit for bit
against a contiguous cache's decode appends (quantised on the host for Q8_0 pools), and what must stay
untouched."""
import ctypes as C

import numpy as np
import pytest

from llmplayer_amd import _lib
from llmplayer_amd import hip_forward_pass as hfp
from llmplayer_amd.paged_batch import PagedKv
from tests import paged_cases as pc

pytestmark = pytest.mark.gpu
F32, I = np.float32, np.int32
MAX_SEQ = 700


def fp(a):
    return None if a is None else a.ctypes.data_as(C.POINTER(C.c_float))


def rotated(x, cos, sin, rope_type, w, eps):
    """x [T][H][D] in 64 bits; cos, sin [T][pairs] or None."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    if cos is None:
        return x
    n = cos.shape[1]
    c, s = cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
    i = np.arange(n)
    one, two = (i, i + n) if rope_type == 2 else (2 * i, 2 * i + 1)
    y = x.copy()
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., one] * s + x[..., two] * c
    return y


def config(handle, hq, hkv, D, rope_type, rope_dim, qw, kw, norm_mode, tables):
    if rope_dim:
        _lib.call("llmp_rope_upload", handle, 0, fp(tables[0]), fp(tables[1]), MAX_SEQ, rope_dim // 2)
    _lib.call("llmp_layer_config", handle, 0, hq, hkv, D, rope_type, 0 if rope_dim else -1, 0, 1, 0.0, 0.0, 1e-6, fp(qw), fp(kw))
    _lib.call("llmp_layer_norm_mode", handle, 0, norm_mode)


CASES = [
    # hq, hkv, D, page, tokens, rope_type, rope_dim, norm, norm_mode, cache, bf16, merged
    (32, 8, 64, 16, 1, 0, 64, False, 0, 0, False, False),
    (32, 8, 64, 16, 37, 0, 64, False, 0, 0, True, True),
    (16, 8, 128, 32, 5, 2, 128, True, 0, 0, False, False),
    (16, 8, 128, 16, 33, 2, 32, True, 0, 0, False, True),
    (24, 8, 96, 64, 9, 2, 96, False, 0, 0, False, False),
    (24, 8, 96, 64, 9, 0, 36, False, 0, 0, True, False),
    (4, 1, 256, 128, 19, 0, 256, True, 0, 0, False, False),
    (8, 2, 256, 256, 6, 2, 256, True, 3, 0, False, False),
    (5, 1, 64, 16, 12, 0, 10, False, 0, 0, False, False),
    (6, 3, 128, 16, 21, 2, 14, False, 0, 0, False, True),
    (32, 8, 64, 16, 3, 0, 0, False, 0, 0, False, False),
    (32, 8, 64, 16, 40, 0, 32, False, 0, 1, False, True),
    (32, 8, 128, 32, 17, 0, 128, False, 0, 2, True, False),
    (16, 8, 128, 16, 11, 2, 128, True, 0, 1, False, False),
    (16, 8, 128, 16, 11, 2, 64, False, 0, 1, False, False),
    (16, 8, 64, 16, 11, 2, 16, False, 0, 2, True, False),
    (8, 2, 256, 64, 4, 0, 64, False, 2, 0, False, False),
    (8, 2, 256, 64, 7, 2, 256, False, 0, 1, False, False),
    (16, 8, 128, 16, 13, 2, 128, False, 0, 2, False, True),
    (16, 8, 128, 16, 13, 2, 48, False, 0, 1, False, False),
    (32, 8, 64, 32, 70, 2, 32, False, 0, 1, True, True),
    (24, 8, 96, 16, 7, 2, 96, False, 0, 1, False, False),
    (24, 8, 96, 16, 7, 2, 64, False, 0, 1, True, False),
    (24, 8, 96, 16, 7, 0, 96, False, 0, 2, False, False),
]


@pytest.mark.parametrize("hq,hkv,D,page,T,rope_type,rope_dim,norm,norm_mode,cache,bf16,merged", CASES)
def test_append(hq, hkv, D, page, T, rope_type, rope_dim, norm, norm_mode, cache, bf16, merged):
    rng = np.random.default_rng(T * 31 + D + rope_dim)
    print(f"[gpu] append {hq}/{hkv}/{D} T={T} rope={rope_dim}/{rope_type} cache={cache}", flush=True)
    tables = hfp.rope_table(rope_dim, MAX_SEQ, 1e5) if rope_dim else None
    qw, kw = ((rng.random(D) + 0.5).astype(F32) for _ in range(2)) if norm else (None, None)
    widths = (hq * D, hkv * D, hkv * D)
    pad = 8 if merged else 0
    rows = rng.standard_normal((T, sum(widths) + pad)).astype(F32) * F32(1.7)
    if bf16:
        raw = hfp.to_bf16(rows).reshape(rows.shape)
        rows = hfp.from_bf16(raw).reshape(rows.shape)
    else:
        raw = rows
    cut = np.cumsum((0,) + widths)
    parts = [rows[:, a:b] for a, b in zip(cut[:-1], cut[1:])]
    n_pages = -(-T // page) + 2
    positions = rng.permutation(MAX_SEQ)[:T].astype(I)
    slots = rng.permutation(n_pages * page)[:T].astype(I)
    with pc.Device() as d:
        kv = PagedKv(1, n_pages, page, MAX_SEQ, hkv, D, cache)
        ref = hfp.KvCache(1, MAX_SEQ, hkv, D)
        try:
            for h in (kv.handle, ref.handle):
                config(h, hq, hkv, D, rope_type, rope_dim, qw, kw, norm_mode, tables)
            empty = {w: (rng.integers(-100, 100, s) if t == np.int8 else rng.standard_normal(s)).astype(t)
                     for w, (s, t) in kv._shapes().items()}
            kv.write(0, empty)
            size = 2 if bf16 else 4
            if merged:
                base, st = d.up(raw), [raw.shape[1]] * 3
                ptr = [base + int(c) * size for c in cut[:3]]
            else:
                ptr = [d.up(raw[:, a:b]) for a, b in zip(cut[:-1], cut[1:])]
                st = list(widths)
            ostride = hq * D + (4 if merged else 0)
            out = d.up(np.full((T + 1, ostride), 77, F32))
            args = (kv.handle, 0, T, d.up(positions), d.up(slots), 1 if bf16 else 0, ptr[0], st[0], ptr[1], st[1], ptr[2], st[2],
                    out, ostride, 0)
            _lib.call("llmp_paged_append", *args)
            got = d.down(out, F32, (T + 1, ostride))
            assert (got[T] == 77).all() and (got[:, hq * D:] == 77).all()
            cs = [None, None] if tables is None else [t[positions] for t in tables]
            want = rotated(parts[0].reshape(T, hq, D), cs[0], cs[1], rope_type, qw, 1e-6)
            # two fp32 products and a sum per value (3 * 2^-24 of the pair's magnitude), and with the
            # norm a sum of D squares, root, reciprocal and two products (D + 6) * 2^-24
            tol = np.abs(want).max(-1, keepdims=True) * np.sqrt(2) * (3 + (D + 6 if norm else 0)) * 2.0 ** -24
            err = np.abs(got[:T, :hq * D].reshape(T, hq, D) - want)
            assert (err <= tol).all(), err.max()
            # the stored rows: one decode append per token into a contiguous cache
            dq, dk, dv, do = (d.up(np.zeros(max(w, 4), F32)) for w in (hq * D, hkv * D, hkv * D, hq * D))
            held = kv.read(0)
            touched = np.zeros(n_pages * page, bool)
            for t in range(T):
                for p, x in zip((dq, dk, dv), parts):
                    x = np.ascontiguousarray(x[t])
                    _lib.call("llmp_memcpy_htod", p, x.ctypes.data, x.nbytes, 0)
                _lib.call("llmp_attn_decode", ref.handle, 0, int(positions[t]), dq, dk, dv, do, 0, 0)
                pg, r = divmod(int(slots[t]), page)
                touched[slots[t]] = True
                if cache == 0:
                    k, v = ref.read(0, int(positions[t]), 1)
                    rk = {"k": k, "v": v}
                else:   # the fp32 rows of a fp32 cache, quantised
                    rk = dict(zip(("k", "v"), ref.read(0, int(positions[t]), 1)))
                    for w in "kv":
                        x = rk[w].reshape(-1, 32)
                        rk[w + "s"] = np.abs(x).max(1) / F32(127) if cache == 2 else np.abs(x).max(1) * F32(1 / 127)
                        with np.errstate(divide="ignore"):
                            y = x * np.where(rk[w + "s"] > 0, F32(1) / rk[w + "s"], F32(0))[:, None]
                        y = np.trunc(y) if cache == 2 else np.floor(y) + (y - np.floor(y) >= F32(0.5))
                        rk[w] = np.clip(y, -128, 127).astype(np.int8)
                for w, x in rk.items():
                    mine = held[w][pg, :, r]
                    assert np.array_equal(mine.reshape(-1).view(np.uint8), np.ascontiguousarray(x).reshape(-1).view(np.uint8)), (t, w)
            for w in held:
                a = held[w].transpose(0, 2, 1, 3).reshape(n_pages * page, -1)[~touched]
                b = empty[w].transpose(0, 2, 1, 3).reshape(n_pages * page, -1)[~touched]
                assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), f"{w}: other rows were written"
        finally:
            kv.destroy()
            ref.destroy()


@pytest.mark.parametrize("D,rope_type,rope_dim,cache,bf16,norm", [
    (64, 0, 64, 0, False, False), (64, 2, 64, 1, True, True), (128, 2, 128, 1, False, False), (128, 0, 64, 2, True, True),
    (96, 0, 96, 1, False, True), (256, 2, 24, 0, True, True), (128, 0, 0, 1, False, False)])
def test_every_alignment_stores_the_same(D, rope_type, rope_dim, cache, bf16, norm):
    """Rows that load in fours and rows at odd strides and offsets: the same bytes out of both."""
    rng = np.random.default_rng(D + rope_dim)
    hq, hkv, page, n_pages, T = 6, 3, 16, 3, 33
    tables = hfp.rope_table(rope_dim, MAX_SEQ, 1e5) if rope_dim else None
    rows = rng.standard_normal((T, (hq + 2 * hkv) * D)).astype(F32)
    raw = hfp.to_bf16(rows).reshape(rows.shape) if bf16 else rows
    positions, slots = rng.permutation(MAX_SEQ)[:T].astype(I), rng.permutation(n_pages * page)[:T].astype(I)
    cut = np.cumsum([0, hq * D, hkv * D, hkv * D])
    qw, kw = ((rng.random(D) + 0.5).astype(F32) for _ in range(2)) if norm else (None, None)
    seen = []
    for pad, first in ((0, 0), (8, 0), (1, 0), (3, 1), (4, 2)):
        with pc.Device() as d:
            kv = PagedKv(1, n_pages, page, MAX_SEQ, hkv, D, cache)
            try:
                config(kv.handle, hq, hkv, D, rope_type, rope_dim, qw, kw, 0, tables)
                kv.write(0, {w: np.zeros(s, t) for w, (s, t) in kv._shapes().items()})
                held = np.zeros((T, raw.shape[1] + pad), raw.dtype)
                held[:, :raw.shape[1]] = raw
                flat = np.concatenate([np.zeros(first, raw.dtype), held.reshape(-1)])
                base, stride, size = d.up(flat) + first * raw.itemsize, held.shape[1], raw.itemsize
                out = d.up(np.zeros((T, hq * D + pad), F32))
                _lib.call("llmp_paged_append", kv.handle, 0, T, d.up(positions), d.up(slots), 1 if bf16 else 0,
                          base, stride, base + int(cut[1]) * size, stride, base + int(cut[2]) * size, stride, out, hq * D + pad, 0)
                got = kv.read(0)
                got["q"] = d.down(out, F32, (T, hq * D + pad))[:, :hq * D]
                seen.append({w: np.ascontiguousarray(x).view(np.uint8) for w, x in got.items()})
            finally:
                kv.destroy()
    for other in seen[1:]:
        assert all(np.array_equal(other[w], seen[0][w]) for w in seen[0])


@pytest.mark.parametrize("norm", [False, True])
def test_tokens_without_position_or_slot(norm):
    """Bad positions skip a token, bad slots store nothing; both leave everything else as it was."""
    rng = np.random.default_rng(3)
    hq, hkv, D, page, n_pages, T = 8, 2, 64, 16, 3, 11
    tables = hfp.rope_table(D, MAX_SEQ, 1e4)
    w = (rng.random(D) + 0.5).astype(F32) if norm else None
    q, k, v = (rng.standard_normal((T, h * D)).astype(F32) for h in (hq, hkv, hkv))
    positions = np.array([0, -1, MAX_SEQ, MAX_SEQ - 1, -2 ** 31, 2 ** 31 - 1, 5, 6, 7, 8, 9], I)
    slots = np.array([3, 4, 5, 47, 6, 7, -1, 48, -2 ** 31, 2 ** 31 - 1, 0], I)
    with pc.Device() as d:
        kv = PagedKv(1, n_pages, page, MAX_SEQ, hkv, D)
        try:
            config(kv.handle, hq, hkv, D, 0, D, w, w, 0, tables)
            empty = {x: rng.standard_normal(s).astype(t) for x, (s, t) in kv._shapes().items()}
            kv.write(0, empty)
            out = d.up(np.full((T, hq * D), 77, F32))
            a = (d.up(q), hq * D, d.up(k), hkv * D, d.up(v), hkv * D, out, hq * D, 0)
            _lib.call("llmp_paged_append", kv.handle, 0, T, d.up(positions), d.up(slots), 0, *a)
            got = d.down(out, F32, (T, hq * D))
            live = [0, 3, 6, 7, 8, 9, 10]
            assert (np.delete(got, live, 0) == 77).all()
            at = positions[live]
            want = rotated(q[live].reshape(-1, hq, D), tables[0][at], tables[1][at], 0, w, 1e-6)
            assert np.abs(got[live].reshape(want.shape) - want).max() < 1e-4
            held = kv.read(0)
            for x in "kv":
                same = (held[x] == empty[x]).all((1, 3)).reshape(-1)
                assert np.flatnonzero(~same).tolist() == [0, 3, 47], x
            # only the queries, in place: same values; the pool stays
            pq = d.up(q)
            _lib.call("llmp_paged_append", kv.handle, 0, T, d.up(positions), 0, 0, pq, hq * D, 0, 0, 0, 0, pq, hq * D, 0)
            mine = d.down(pq, F32, (T, hq * D))
            assert np.array_equal(mine[live], got[live]) and np.array_equal(np.delete(mine, live, 0), np.delete(q, live, 0))
            again = kv.read(0)
            assert all(np.array_equal(again[x], held[x]) for x in held)
        finally:
            kv.destroy()
