"""GPU checks of llmp_paged_tables against the sequence-by-sequence reference: every array exactly."""
import ctypes as C

import numpy as np
import pytest

from llmplayer_amd import _lib
from llmplayer_amd.paged_batch import PagedKv
from tests import paged_cases as pc

pytestmark = pytest.mark.gpu
I = np.int32


def make(rng, n, page, max_seq, shared, most_new, ended, extra_pages=7):
    """Lengths and tables of n sequences, and a free list."""
    low = shared * page
    length = rng.integers(low, max_seq - most_new + 1, n).astype(I)
    length[rng.random(n) < 0.2] = low
    grow = rng.integers(0, most_new + 1, n).astype(I)
    grow[rng.random(n) < 0.2] = 0
    grow[rng.random(n) < ended] = -1 - rng.integers(0, 3)
    up = lambda x: -(-x // page)  # noqa: E731
    width = up(max_seq)
    total = shared + int(sum(up(int(a) + max(int(g), 0)) for a, g in zip(length, grow))) + extra_pages
    order = (rng.permutation(total - shared) + shared).astype(I)
    blocks = np.full((n, width), -5, I)
    blocks[:, :shared] = np.arange(shared)
    at = 0
    for b in range(n):
        have = up(int(length[b]))
        blocks[b, shared:have] = order[at:at + max(have - shared, 0)]
        at += max(have - shared, 0)
    free = np.full(total, -7, I)
    n_free = total - shared - at
    free[:n_free] = order[at:]
    return {"length": length, "grow": grow, "free": free, "n_free": n_free, "blocks": blocks, "n_pages": total}


def run(d, kv, c, shared, max_tokens, in_place=False, before=None, stream=0):
    n = len(c["length"])
    p = {"len": d.up(c["length"]), "grow": d.up(c["grow"]), "free": d.up(c["free"]),
         "n_free": d.up(np.array([c["n_free"]], I)), "blocks": d.up(c["blocks"])}
    p["len_out"] = p["len"] if in_place else d.up(np.full(n, 99, I))
    p["n_free_out"] = p["n_free"] if in_place else d.up(np.full(1, 99, I))
    p["seq_start"] = d.up(np.full(n + 1, 99, I))
    p["positions"], p["slots"] = d.up(np.full(max_tokens + 1, 99, I)), d.up(np.full(max_tokens + 1, 99, I))
    p["status"] = d.up(np.full(1, 99, I))
    args = ("llmp_paged_tables", kv.handle, n, shared, max_tokens, p["len"], p["grow"], p["free"], p["n_free"], p["blocks"],
            p["len_out"], p["n_free_out"], p["seq_start"], p["positions"], p["slots"], p["status"], stream)
    _lib.call(*args)
    return p, args


def check(d, p, c, want, max_tokens, what):
    n = len(c["length"])
    got = {"status": d.down(p["status"], I, 1)[0], "n_free": d.down(p["n_free_out"], I, 1)[0],
           "seq_start": d.down(p["seq_start"], I, n + 1), "len": d.down(p["len_out"], I, n),
           "positions": d.down(p["positions"], I, max_tokens + 1), "slots": d.down(p["slots"], I, max_tokens + 1),
           "blocks": d.down(p["blocks"], I, c["blocks"].shape), "free": d.down(p["free"], I, c["free"].shape)}
    for w in got:
        if w in ("positions", "slots"):
            assert got[w][max_tokens] == 99, f"{what}: {w} written past its end"
            got[w] = got[w][:max_tokens]
        assert np.array_equal(got[w], want[w]), (what, w, np.argwhere(np.asarray(got[w] != want[w]))[:4].tolist())


@pytest.mark.parametrize("in_place", [False, True], ids=["", "in_place"])
@pytest.mark.parametrize("n,page,shared,most_new,ended", [
    (1, 16, 0, 1, 0), (1, 16, 0, 0, 0), (1, 16, 0, 70, 0), (2, 16, 1, 1, 1), (3, 64, 2, 200, 0.4), (63, 16, 0, 1, 0.1), (64, 32, 3, 5, 0.2),
    (65, 256, 1, 40, 0.2), (1023, 16, 1, 1, 0.1), (1025, 16, 0, 3, 0.3), (4096, 64, 3, 4, 0.1), (8192, 128, 0, 1, 0.05),
    (40, 16, 2, 900, 0.3)])
def test_tables(n, page, shared, most_new, ended, in_place):
    rng = np.random.default_rng(n * 7 + page)
    max_seq = max(page * (shared + 3) + 5, most_new + page * shared + 17, 700 if n < 200 else 0)
    c = make(rng, n, page, max_seq, shared, most_new, ended)
    max_tokens = int(np.maximum(c["grow"], 0).sum()) + (n % 3)
    max_tokens = max(max_tokens, 1)
    print(f"[gpu] tables n={n} page={page} tokens={max_tokens}", flush=True)
    want = pc.reference_tables(c["length"], c["grow"], c["free"], c["n_free"], c["blocks"], page, max_seq, shared, max_tokens,
                               c["n_pages"])
    assert want["status"] == 0
    kv = None
    with pc.Device() as d:
        kv = PagedKv(1, c["n_pages"], page, max_seq, 1, 64)
        try:
            p, _ = run(d, kv, c, shared, max_tokens, in_place)
            check(d, p, c, want, max_tokens, "tables")
        finally:
            kv.destroy()


@pytest.mark.parametrize("what", ["short", "no_pages", "too_long", "negative", "tokens", "free_count", "free_negative", "returned_twice"])
@pytest.mark.parametrize("in_place", [False, True], ids=["", "in_place"])
def test_refused_steps_change_nothing(what, in_place):
    rng = np.random.default_rng(5)
    page, shared, max_seq = 16, 1, 500
    c = make(rng, 70, page, max_seq, shared, 40, 0.2, extra_pages=0)
    max_tokens = int(np.maximum(c["grow"], 0).sum())
    if what in ("short", "no_pages"):
        c["grow"] = np.abs(c["grow"])
        max_tokens = int(c["grow"].sum())
        c["n_free"] = c["n_free"] - 1 if what == "short" else 0
        need = sum(-(-int(a + g) // page) + -int(a) // page for a, g in zip(c["length"], c["grow"]))
        c["n_free"] = need - 1 if what == "short" else 0
    elif what == "too_long":
        c["length"][69], c["grow"][69] = max_seq, 1
    elif what == "negative":
        c["length"][3] = -4
    elif what == "tokens":
        max_tokens -= 1
    elif what == "free_count":
        c["n_free"] = c["n_pages"] + 1
    elif what == "free_negative":
        c["n_free"] = -1
    else:
        c["n_free"], c["grow"] = c["n_pages"], np.full(70, -1, I)
    want = pc.reference_tables(c["length"], c["grow"], c["free"], c["n_free"], c["blocks"], page, max_seq, shared, max_tokens,
                               c["n_pages"])
    assert want["status"] != 0
    with pc.Device() as d:
        kv = PagedKv(1, c["n_pages"], page, max_seq, 1, 64)
        try:
            p, _ = run(d, kv, c, shared, max_tokens, in_place)
            check(d, p, c, want, max_tokens, what)
        finally:
            kv.destroy()


@pytest.mark.parametrize("n", [4096, 4095])
def test_sums_beyond_32_bits(n):
    """2^20 new tokens of each of 4096 sequences: 2^32 of them."""
    max_seq, page = 1 << 20, 256
    c = {"length": np.zeros(n, I), "grow": np.full(n, 1 << 20, I), "free": np.arange(8, dtype=I), "n_free": 8,
         "blocks": np.full((n, max_seq // page), -1, I), "n_pages": 8}
    with pc.Device() as d:
        kv = PagedKv(1, 8, page, max_seq, 1, 64)
        try:
            p, _ = run(d, kv, c, 0, 1000)
            want = {"status": -2, "n_free": 8, "len": c["length"], "seq_start": np.zeros(n + 1, I), "positions": np.full(1000, -1, I),
                    "slots": np.full(1000, -1, I), "blocks": c["blocks"], "free": c["free"]}
            check(d, p, c, want, 1000, "2^32 tokens")
        finally:
            kv.destroy()


def test_entries_outside_the_pool_give_no_slot():
    c = {"length": np.array([20, 5], I), "grow": np.array([3, 1], I), "free": np.arange(6, dtype=I), "n_free": 4,
         "blocks": np.array([[4, 77, -1, -1], [-3, 0, 0, 0]], I), "n_pages": 6}
    want = pc.reference_tables(c["length"], c["grow"], c["free"], 4, c["blocks"], 16, 64, 0, 6, 6)
    assert want["slots"].tolist() == [-1] * 6 and want["positions"].tolist() == [20, 21, 22, 5, -1, -1]
    with pc.Device() as d:
        kv = PagedKv(1, 6, 16, 64, 1, 64)
        try:
            p, _ = run(d, kv, c, 0, 6)
            check(d, p, c, want, 6, "bad pages")
        finally:
            kv.destroy()


def test_captured_steps_advance_in_place():
    """One captured step, replayed as the sequences grow, between eager steps on another handle."""
    rng = np.random.default_rng(11)
    page, n, max_seq = 16, 300, 400
    c = make(rng, n, page, max_seq, 1, 3, 0.0, extra_pages=900)
    c["length"] = np.minimum(c["length"], 330).astype(I)
    other = make(rng, 2000, page, 100, 0, 2, 0.2)
    with pc.Device() as d:
        kv, kv2 = PagedKv(1, c["n_pages"], page, max_seq, 1, 64), PagedKv(1, other["n_pages"], page, 100, 1, 64)
        try:
            max_tokens = 3 * n
            st = C.c_uint64()
            _lib.call("llmp_stream_create", C.byref(st))
            g = C.c_uint64()
            state = {k: (v.copy() if isinstance(v, np.ndarray) else v) for k, v in c.items()}
            p, args = run(d, kv, c, 1, max_tokens, in_place=True, stream=st.value)
            _lib.call("llmp_stream_sync", st.value)
            _lib.call("llmp_graph_begin", st.value)
            _lib.call(*args)
            _lib.call("llmp_graph_end", st.value, C.byref(g))
            for step in range(6):
                want = pc.reference_tables(state["length"], state["grow"], state["free"], state["n_free"], state["blocks"], page,
                                           max_seq, 1, max_tokens, c["n_pages"])
                check(d, p, c, want, max_tokens, f"step {step}")
                state.update(length=want["len"], free=want["free"], n_free=want["n_free"], blocks=want["blocks"])
                state["grow"] = rng.integers(-1 if step == 3 else 0, 4, n).astype(I)
                _lib.call("llmp_memcpy_htod", p["grow"], state["grow"].ctypes.data, state["grow"].nbytes, st.value)
                _lib.call("llmp_graph_launch", g.value, st.value)
                p2, _ = run(d, kv2, other, 0, 4000)
                _lib.call("llmp_stream_sync", st.value)
                _lib.call("llmp_stream_sync", 0)
            _lib.call("llmp_graph_destroy", g.value)
            _lib.call("llmp_stream_destroy", st.value)
        finally:
            kv.destroy()
            kv2.destroy()


def test_handles_refuse_each_others_calls():
    with pc.Device() as d:
        kv = PagedKv(1, 4, 16, 64, 1, 64)
        h = C.c_uint64()
        _lib.call("llmp_kv_create", 1, 64, 1, 64, 0, C.byref(h))
        try:
            x = d.up(np.zeros(64 * 16, np.float32))
            assert _lib.status("llmp_attn_decode", kv.handle, 0, 0, x, x, x, x, 0, 0) == 1
            assert _lib.status("llmp_attn_prefill_f32", kv.handle, 0, 0, 2, x, x, x, 0, x, 0) == 1
            assert _lib.status("llmp_kv_clear", kv.handle, 0) == 1
            assert _lib.status("llmp_kv_read", kv.handle, 0, 0, 1, None, None) == 1
            assert _lib.status("llmp_block_config", kv.handle, 64, 0.0) == 1
            n = C.c_uint64()
            assert _lib.status("llmp_paged_bytes", h.value, C.byref(n)) == 1
            assert _lib.status("llmp_paged_bind", h.value, x) == 1
            assert _lib.status("llmp_paged_attn", h.value, 0, 1, 1, 0, 0, x, x, x, x, 64, 0, x, 64, 0) == 1
            assert _lib.status("llmp_paged_bytes", 1 << 40, C.byref(n)) == 8
            # a pool that is not bound, a layer that is not configured, a pool that is not aligned
            _lib.call("llmp_paged_create", 1, 4, 16, 64, 1, 64, 0, C.byref(n))
            assert _lib.status("llmp_paged_attn", kv.handle, 0, 1, 1, 0, 0, x, x, x, x, 64, 0, x, 64, 0) == 1
            assert _lib.status("llmp_paged_attn", kv.handle, 1, 1, 1, 0, 0, x, x, x, x, 64, 0, x, 64, 0) == 2
            _lib.call("llmp_layer_config", n.value, 0, 1, 1, 64, 0, -1, 0, 1, 0.0, 0.0, 1e-6, None, None)
            assert _lib.status("llmp_paged_attn", n.value, 0, 1, 1, 0, 0, x, x, x, x, 64, 0, x, 64, 0) == 1
            assert "llmp_paged_bind" in _lib.last_error()
            assert _lib.status("llmp_paged_bind", n.value, x + 16) == 1
            assert _lib.status("llmp_paged_planes", n.value, 0, None, None, None, None) == 1
            _lib.call("llmp_kv_destroy", n.value)
        finally:
            kv.destroy()
            _lib.call("llmp_kv_destroy", h.value)
