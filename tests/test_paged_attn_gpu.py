"""GPU checks of llmp_paged_attn against attention in 64 bits over the same pages."""
import numpy as np
import pytest

from llmplayer_amd import _lib
from llmplayer_amd.paged_batch import PagedKv
from tests import paged_cases as pc

pytestmark = pytest.mark.gpu
F32, I = np.float32, np.int32


class Batch:
    """Sequences of given rows and new tokens over a shuffled pool; what no sequence holds is garbage."""

    def __init__(self, rng, hq, hkv, D, page, prefix, held, new, cache=0, window=0, pad=0, garbage="nan", size=(2.0, 1.0),
                 extra_pages=2, spread=0):
        self.hq, self.hkv, self.D, self.page, self.prefix, self.window, self.cache = hq, hkv, D, page, prefix, window, cache
        total = [prefix + h + n for h, n in zip(held, new)]
        self.max_seq = max(max(total), 1) + 3
        up = lambda x: -(-x // page)  # noqa: E731
        whole, width = prefix // page, up(self.max_seq)
        self.n_pages = up(prefix) + sum(up(t) - whole for t in total) + extra_pages
        order = rng.permutation(self.n_pages).astype(I)
        self.blocks = np.full((len(held), width), -1, I)
        at = whole
        for b, t in enumerate(total):
            self.blocks[b, :whole] = order[:whole]
            self.blocks[b, whole:up(t)] = order[at:at + up(t) - whole]
            at += up(t) - whole
        self.total, self.T = total, sum(new)
        self.seq_start = np.concatenate([[0], np.cumsum(new)]).astype(I)
        self.positions = np.concatenate([np.arange(t - n, t) for t, n in zip(total, new)] + [np.full(pad, -1)]).astype(I)
        self.n_tokens = self.T + pad
        self.q = rng.standard_normal((self.n_tokens, hq, D)).astype(F32)
        shape = (self.n_pages, hkv, page, D)
        used = np.zeros((self.n_pages, page), bool)
        for b, t in enumerate(total):
            j = np.arange(t)
            own = np.where(j < prefix, self.blocks[0][j // page], self.blocks[b][j // page])
            used[own, j % page] = True
        used = used[:, None, :, None]
        if cache == 0:
            self.planes = {w: (rng.standard_normal(shape) * s).astype(F32) for w, s in zip("kv", size)}
            if spread:   # magnitudes that differ by 2^spread between rows
                for w in "kv":
                    self.planes[w] *= np.exp2(rng.integers(-spread, 1, (self.n_pages, 1, page, 1))).astype(F32)
            bad = {"nan": np.nan, "inf": np.inf, "huge": 3e38}[garbage]
            for w in "kv":
                self.planes[w] = np.where(used, self.planes[w], F32(bad))
        else:
            self.planes = {}
            for w, s in zip("kv", size):
                self.planes[w] = rng.integers(-127, 128, shape).astype(np.int8)
                sc = ((rng.random(shape[:3] + (D // 32,)) + 0.5) * s / 73).astype(F32)
                bad = {"nan": np.nan, "inf": np.inf, "huge": 3e38}[garbage]
                self.planes[w + "s"] = np.where(used, sc, F32(bad))

    def run(self, d, scale=0.0, softcap=0.0, sinks=None, gate=None, max_len=0, kv=None, out_fill=77.0, prefix=None, strides=0,
            stream=0, blocks=None, positions=None):
        own = kv is None
        if own:
            kv = PagedKv(1, self.n_pages, self.page, self.max_seq, self.hkv, self.D, self.cache)
        try:
            pc.layer_config(kv, self.hq, window=self.window, scale=scale, softcap=softcap)
            if sinks is not None:
                import ctypes as C
                _lib.call("llmp_layer_sinks", kv.handle, 0, sinks.ctypes.data_as(C.POINTER(C.c_float)))
            kv.write(0, self.planes)
            w = self.hq * self.D
            q = np.full((self.n_tokens, w + strides), np.nan, F32)
            q[:, :w] = self.q.reshape(self.n_tokens, w)
            out = d.up(np.full((self.n_tokens, w + 2 * strides), out_fill, F32))
            self.args = (kv.handle, 0, len(self.seq_start) - 1, self.n_tokens, self.prefix if prefix is None else prefix, max_len,
                         d.up(self.seq_start), d.up(self.positions if positions is None else positions),
                         d.up(self.blocks if blocks is None else blocks), d.up(q), w + strides, 0 if gate is None else d.up(gate),
                         out, w + 2 * strides, stream)
            _lib.call("llmp_paged_attn", *self.args)
            got = d.down(out, F32, (self.n_tokens, w + 2 * strides))
            assert (got[:, w:] == out_fill).all(), "columns behind the rows were written"
            return got[:, :w].reshape(self.n_tokens, self.hq, self.D)
        finally:
            if own:
                kv.destroy()

    def want(self, **kw):
        blocks, positions, prefix = kw.pop("blocks", self.blocks), kw.pop("positions", self.positions), kw.pop("prefix", self.prefix)
        return pc.reference_attention(self.planes, blocks, self.seq_start, positions, self.q, self.n_tokens, prefix,
                                      self.page, self.max_seq, window=self.window, **kw)

    def check(self, got, want, tol, what=""):
        live = ~np.isnan(want).all((1, 2))
        assert (got[~live] == 77).all(), f"{what}: rows behind the last sequence were written"
        err = np.abs(got[live].astype(np.float64) - want[live])
        assert np.isfinite(got[live]).all(), f"{what}: not finite"
        worst = (err / tol[live].clip(1e-300)).max() if live.any() else 0
        print(f"[gpu] {what}: error {err.max() if live.any() else 0:.2e}, {worst:.2f} of the bound", flush=True)
        assert (err <= tol[live]).all(), (what, err.max(), worst)


def rng_of(*x):
    return np.random.default_rng(sum((i + 1) * int(v * 8) for i, v in enumerate(x)))


SHAPES = [(32, 8, 64), (16, 8, 128), (24, 8, 96), (4, 1, 256), (6, 6, 64), (48, 2, 128), (7, 1, 64), (16, 1, 256)]


@pytest.mark.parametrize("cache", [0, 1], ids=["f32", "q8"])
@pytest.mark.parametrize("hq,hkv,D", SHAPES)
def test_shapes(hq, hkv, D, cache):
    rng = rng_of(hq, hkv, D, cache)
    for page, prefix, held, new in ((16, 50, [0, 1, 30, 100], [1, 1, 1, 1]), (64, 97, [3, 0, 70], [5, 1, 20])):
        b = Batch(rng, hq, hkv, D, page, prefix, held, new, cache)
        with pc.Device() as d:
            b.check(b.run(d), *b.want(), what=f"{hq}/{hkv}/{D} page {page}")


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 31, 32, 33, 64, 257, 1500])
@pytest.mark.parametrize("held,new", [([0], [1]), ([0, 0, 5], [1, 0, 2]), ([31, 32, 33, 700], [1, 1, 1, 1]), ([2, 90], [40, 7])])
def test_prefix_lengths(prefix, held, new):
    rng = rng_of(prefix, len(held), held[-1])
    b = Batch(rng, 8, 2, 64, 16, prefix, held, new, pad=2)
    with pc.Device() as d:
        b.check(b.run(d), *b.want(), what=f"prefix {prefix} held {held}")


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("garbage", ["nan", "inf", "huge"])
@pytest.mark.parametrize("cache", [0, 2], ids=["f32", "q8"])
def test_what_no_sequence_holds_does_not_count(page, garbage, cache):
    rng = rng_of(page, len(garbage), cache)
    b = Batch(rng, 8, 2, 128, page, 77, [1, 19, 260, 0], [1, 3, 1, 17], cache, garbage=garbage, pad=1)
    with pc.Device() as d:
        b.check(b.run(d), *b.want(), what=f"page {page} {garbage}")


@pytest.mark.parametrize("window", [1, 16, 100, 512])
@pytest.mark.parametrize("hq,hkv,D", [(4, 1, 256), (8, 2, 64)])
def test_windows(window, hq, hkv, D):
    rng = rng_of(window, D)
    for prefix, held, new in ((300, [0, 3, 900], [1, 1, 1]), (90, [0, 40, 400], [9, 30, 3])):
        b = Batch(rng, hq, hkv, D, 16, prefix, held, new, window=window, garbage="inf")
        with pc.Device() as d:
            b.check(b.run(d), *b.want(), what=f"window {window} prefix {prefix}")


def test_scale_softcap_sinks_gate():
    rng = rng_of(4)
    b = Batch(rng, 8, 2, 64, 16, 130, [0, 60, 3], [1, 4, 1], pad=1)
    sinks = rng.standard_normal(8).astype(F32) * F32(3)
    gate = rng.standard_normal((b.n_tokens, 8, 64)).astype(F32)
    with pc.Device() as d:
        for kw in ({"scale": 0.3}, {"softcap": 20.0}, {"sinks": sinks}, {"gate": gate},
                   {"scale": 0.2, "softcap": 5.0, "sinks": sinks, "gate": gate}):
            b.check(b.run(d, **kw), *b.want(**kw), what=str(sorted(kw)))


@pytest.mark.parametrize("size", [(1e-6, 1e-8), (3e4, 1e5), (1e-3, 1e30), (1.0, 1e-30), (1e15, 1.0), (1e-20, 1.0)])
def test_magnitudes(size):
    """The bound is relative to the largest values: no magnitude loses the parts' bits."""
    rng = rng_of(len(str(size)))
    b = Batch(rng, 8, 2, 64, 16, 70, [0, 33], [1, 5], size=size)
    b.q *= F32(1 / size[0]) if size[0] < 1 or size[0] > 10 else F32(1)
    with pc.Device() as d:
        b.check(b.run(d), *b.want(), what=f"K {size[0]} V {size[1]}")


def test_rows_of_different_magnitude():
    rng = rng_of(9)
    b = Batch(rng, 8, 2, 128, 16, 200, [0, 33, 200], [1, 5, 1], spread=12)
    with pc.Device() as d:
        b.check(b.run(d), *b.want(), what="spread 2^12")


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_bad_row_spoils_only_the_tokens_that_attend_it(value, where):
    """Token 6 of sequence 1's nine new ones holds it: tokens 0 to 5 and the other sequences do not
    attend it, tokens 6 to 8 do."""
    rng = rng_of(12)
    b = Batch(rng, 8, 2, 64, 16, 40, [0, 21, 50], [2, 9, 3])
    want, tol = b.want()
    p = 40 + 21 + 6
    b.planes[where][b.blocks[1][p // 16], :, p % 16, 5] = value
    with pc.Device() as d:
        got = b.run(d)
    hit = slice(2 + 6, 2 + 9)
    assert not np.isfinite(got[hit][..., 5]).any()
    got[hit], want[hit] = 0, 0
    b.check(got, want, tol, what=f"{value} in {where}")
    # in the prefix, before the window of the later tokens
    b = Batch(rng, 8, 2, 64, 16, 40, [0, 21], [1, 9], window=32)
    want, tol = b.want()
    b.planes[where][b.blocks[0][0], :, 10, 5] = value     # row 10: in the window of positions up to 41
    with pc.Device() as d:
        got = b.run(d)
    assert not np.isfinite(got[0][..., 5]).any()
    got[0], want[0] = 0, 0
    b.check(got, want, tol, what=f"{value} in {where} of the prefix")


def test_blocks_outside_the_pool_hold_no_rows():
    rng = rng_of(14)
    b = Batch(rng, 8, 2, 64, 16, 64, [0, 40], [1, 3])
    blocks = b.blocks.copy()
    blocks[0, 1], blocks[1, 5], blocks[1, 4] = -1, b.n_pages, 2 ** 31 - 1
    blocks[1, 0] = -9      # the prefix is sequence 0's
    with pc.Device() as d:
        b.check(b.run(d, blocks=blocks), *b.want(blocks=blocks), what="bad blocks")
        # nothing at all to attend: zeros, with and without a sink
        none = np.full_like(blocks, -1)
        assert (b.run(d, blocks=none) == 0).all()
        assert (b.run(d, blocks=none, sinks=np.ones(8, F32)) == 0).all()


def test_positions_that_are_none():
    rng = rng_of(15)
    b = Batch(rng, 8, 2, 64, 16, 30, [0, 40], [2, 3])
    positions = b.positions.copy()
    positions[[1, 3]] = -1, b.max_seq
    with pc.Device() as d:
        got = b.run(d, positions=positions)
        b.check(got, *b.want(positions=positions), what="bad positions")
        assert (got[[1, 3]] == 0).all()


def test_no_sequence_holds_tokens():
    rng = rng_of(16)
    b = Batch(rng, 8, 2, 64, 16, 30, [0, 40], [0, 0], pad=5)
    with pc.Device() as d:
        assert (b.run(d) == 77).all()


def test_strides_and_bounds():
    """Rows further apart than they are wide; bounds of the lengths that are too low or high change
    nothing but the order of sums."""
    rng = rng_of(17)
    b = Batch(rng, 8, 2, 96, 32, 300, [0, 900, 5], [1, 1, 6])
    with pc.Device() as d:
        for max_len in (0, 1, 310, b.max_seq):
            b.check(b.run(d, strides=12, max_len=max_len), *b.want(), what=f"max_len {max_len}")
        # no prefix named: the same rows through the tables, whose own blocks hold the prefix's last rows
        for w in "kv":
            for x in b.blocks[1:, 300 // 32]:
                b.planes[w][x, :, :300 % 32] = b.planes[w][b.blocks[0, 300 // 32], :, :300 % 32]
        b.check(b.run(d, prefix=0), *b.want(), what="prefix not named")


@pytest.mark.parametrize("n", [63, 64, 65, 200, 1000])
def test_many_sequences(n):
    rng = rng_of(n)
    held, new = rng.integers(0, 60, n).tolist(), rng.integers(0, 3, n).tolist()
    new[-1] = 1
    b = Batch(rng, 8, 2, 64, 16, 33, held, new)
    with pc.Device() as d:
        b.check(b.run(d), *b.want(), what=f"{n} sequences")


def test_rows_far_into_a_large_pool():
    """Pages whose offsets pass 2^32 bytes (and 2^31 elements in the int8 pool)."""
    import ctypes as C
    rng = rng_of(21)
    for cache, n_pages in ((0, 1200000 // 16), (1, 2400000 // 16)):
        hq, hkv, D, page = 8, 8, 128, 16
        b = Batch(rng, hq, hkv, D, page, 40, [0, 50], [1, 2], cache)
        small, b.n_pages = b.n_pages, n_pages
        assert n_pages * page * hkv * D * (4 if cache == 0 else 1) > 2 ** 32 // (1 if cache == 0 else 2)
        with pc.Device() as d:
            kv = PagedKv(1, n_pages, page, b.max_seq, hkv, D, cache)
            try:
                pc.layer_config(kv, hq)
                at = dict(zip(("k", "ks", "v", "vs"), kv.planes(0)))
                for w, x in b.planes.items():   # the batch's pages as the pool's last ones
                    x = np.ascontiguousarray(x)
                    off = (n_pages - small) * (x.nbytes // small)
                    _lib.call("llmp_memcpy_htod", at[w] + off, x.ctypes.data, x.nbytes, 0)
                blocks = np.where(b.blocks >= 0, b.blocks + n_pages - small, -1).astype(I)
                out = d.up(np.zeros((3, hq, D), F32))
                _lib.call("llmp_paged_attn", kv.handle, 0, 2, 3, 40, 0, d.up(b.seq_start), d.up(b.positions), d.up(blocks),
                          d.up(b.q), hq * D, 0, out, hq * D, 0)
                b.check(d.down(out, F32, (3, hq, D)), *b.want(), what=f"large pool, cache {cache}")
            finally:
                kv.destroy()


@pytest.mark.parametrize("seed", range(48))
def test_drawn(seed):
    """Every shape, cache, page and mask with every other, up to prompts that take items of 128 rows."""
    rng = np.random.default_rng(1000 + seed)
    hq, hkv, D = SHAPES[rng.integers(len(SHAPES))]
    n = int(rng.choice([1, 2, 3, 9, 30]))
    most = int(rng.choice([1, 1, 4, 40, 130])) if n < 30 else 2
    prefix = int(rng.choice([0, 1, 47, 64, 200, 777]))
    held = rng.integers(0, int(rng.choice([1, 40, 600])), n).tolist()
    new = rng.integers(0, most + 1, n).tolist()
    new[int(rng.integers(n))] = most
    b = Batch(rng, hq, hkv, D, int(rng.choice([16, 32, 64, 128, 256])), prefix, held, new, cache=int(rng.integers(3)),
              window=int(rng.choice([0, 0, 0, 1, 50, 300])), pad=int(rng.integers(3)),
              garbage=str(rng.choice(["nan", "inf", "huge"])))
    kw = {}
    if rng.random() < 0.3:
        kw["scale"] = 0.2
    if rng.random() < 0.3:
        kw["softcap"] = 10.0
    if rng.random() < 0.3:
        kw["sinks"] = rng.standard_normal(hq).astype(F32)
    if rng.random() < 0.3:
        kw["gate"] = rng.standard_normal((b.n_tokens, hq, D)).astype(F32)
    if rng.random() < 0.25:     # tokens anywhere in their sequences, and none
        positions = b.positions.copy()
        for s, t in enumerate(b.total):
            for i in range(b.seq_start[s], b.seq_start[s + 1]):
                positions[i] = rng.integers(-1, t)
        kw["positions"] = positions
    if rng.random() < 0.25:     # blocks that no page holds
        blocks = b.blocks.copy()
        blocks[rng.random(blocks.shape) < 0.1] = rng.choice([-1, b.n_pages, 2 ** 31 - 1, -2 ** 31])
        kw["blocks"] = blocks
    with pc.Device() as d:
        got = b.run(d, strides=4 * int(rng.integers(3)), max_len=int(rng.choice([0, 1, b.max_seq])), **kw)
        b.check(got, *b.want(**kw), what=f"seed {seed}: {hq}/{hkv}/{D} n {n} new {most} prefix {prefix} cache {b.cache} {sorted(kw)}")


@pytest.mark.parametrize("cache", [0, 1], ids=["f32", "q8"])
@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 64), (8, 2, 96), (8, 2, 128), (4, 1, 256)])
def test_a_bad_row_among_many_queries(hq, hkv, D, cache):
    """Row 75 of a prompt of 150 tokens: the tokens before it stay what they were."""
    rng = rng_of(hq, D, cache, 30)
    b = Batch(rng, hq, hkv, D, 32, 45, [0, 10], [150, 90], cache)
    want, tol = b.want()
    p = 45 + 75
    for w in (("k", "v") if cache == 0 else ("ks", "vs")):
        for value in (np.nan, np.inf):
            plane = b.planes[w]
            kept = plane.copy()
            plane[b.blocks[0][p // 32], :, p % 32, 0] = value
            with pc.Device() as d:
                got = b.run(d)
            b.planes[w][:] = kept
            hit = slice(75, 150)
            assert not np.isfinite(got[hit][..., 0]).any(), (w, value)
            y = want.copy()
            got[hit], y[hit] = 0, 0
            b.check(got, y, tol, what=f"{value} in {w}")


def test_other_streams():
    """The same call on a stream of its own, and twice on one handle in turn on two streams."""
    import ctypes as C
    rng = rng_of(31)
    b = Batch(rng, 8, 2, 128, 16, 300, [0, 90, 5], [1, 3, 60])
    kv = PagedKv(1, b.n_pages, b.page, b.max_seq, b.hkv, b.D, 0)
    streams = [C.c_uint64() for _ in range(2)]
    try:
        for s in streams:
            _lib.call("llmp_stream_create", C.byref(s))
        with pc.Device() as d:
            first = b.run(d, kv=kv)
            b.check(first, *b.want(), what="library stream")
            for s in streams + streams:
                out = d.up(np.full((b.n_tokens, b.hq * b.D), 77, F32))
                args = list(b.args)
                args[12], args[14] = out, s.value
                _lib.call("llmp_paged_attn", *args)
                _lib.call("llmp_stream_sync", s.value)
                assert np.array_equal(d.down(out, F32, first.shape).view(np.uint32), first.view(np.uint32))
    finally:
        for s in streams:
            _lib.call("llmp_stream_destroy", s.value)
        kv.destroy()
