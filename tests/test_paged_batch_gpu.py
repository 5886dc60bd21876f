"""The paged batch as it is used: HipBatchPass against one contiguous cache per sequence
(HipForwardPass), through a prefix, steps of different lengths, ended and new sequences, and the same
steps captured and replayed."""
import ctypes as C

import numpy as np
import pytest

from llmplayer_amd import _lib
from llmplayer_amd import hip_forward_pass as hfp
from llmplayer_amd.paged_batch import HipBatchPass
from tests import paged_cases as pc

pytestmark = pytest.mark.gpu
F32, I = np.float32, np.int32

CONFIGS = {
    "llama": hfp.ModelConfig(8, 2, 64, 2, architecture=hfp.ARCH_LLAMA, rope_freq_base=500000.0),
    "qwen3": hfp.ModelConfig(16, 8, 128, 2, architecture=hfp.ARCH_QWEN3, rope_freq_base=1e6),
    "gemma3": hfp.ModelConfig(4, 1, 256, 6, architecture=hfp.ARCH_GEMMA3, rope_freq_base=1e6, sliding_window=48),
}


def qk_norm(c, rng):
    if c.architecture == hfp.ARCH_LLAMA:
        return None
    return [tuple((rng.random(c.head_size) + 0.5).astype(F32) for _ in range(2)) for _ in range(c.block_count)]


def step_inputs(rng, c, n):
    return [[rng.standard_normal((n, w)).astype(F32) for w in (c.q_dim, c.kv_dim, c.kv_dim)] for _ in range(c.block_count)]


def upload(d, c, rows, max_tokens):
    """Device projections padded to max_tokens rows (what pads them is never used)."""
    out = []
    for x in rows:
        p = np.full((max_tokens, x.shape[1]), np.nan, F32)
        p[:len(x)] = x
        out.append(d.up(p))
    return out


class Single:
    """The same sequence in a contiguous cache of its own."""

    def __init__(self, c, max_seq, norm, dtype, prefix_rows):
        self.fp, self.len = hfp.HipForwardPass(c, max_seq, qk_norm=norm, kv_dtype=dtype), 0
        for part in prefix_rows:
            self.step(part)

    def step(self, rows):
        """rows: per layer (q, k, v) of the new tokens, one decode each."""
        c, n = self.fp.config, len(rows[0][0])
        out = np.zeros((c.block_count, n, c.q_dim), F32)
        st = hfp.InferenceState.create(c)
        for t in range(n):
            for layer, (q, k, v) in enumerate(rows):
                st.q[:], st.k[:], st.v[:] = q[t], k[t], v[t]
                self.fp.forwardAttentionOnly(st, layer, self.len + t)
                out[layer, t] = st.xb2
        self.len += n
        return out


@pytest.mark.parametrize("name,dtype", [("llama", 0), ("llama", 1), ("qwen3", 0), ("qwen3", 2), ("gemma3", 0)])
def test_batch_matches_single_sequences(name, dtype):
    c = CONFIGS[name]
    rng = np.random.default_rng(len(name) + dtype)
    norm, max_seq, page, prefix, seqs, max_tokens = qk_norm(c, rng), 160, 16, 48, 5, 40
    parts = [step_inputs(rng, c, 30), step_inputs(rng, c, 18)]
    steps = [[7, 1, 0, 30, 2], [1, 1, 1, 1, 1], [1, 1, 1, 1, 1], [3, -1, 9, 1, -1], [1, 12, 1, 1, 5], [1, 1, 1, 1, 1]]
    singles = [Single(c, max_seq, norm, dtype, parts) for _ in range(seqs)]
    kvd = singles[0].fp
    with pc.Device() as d, HipBatchPass(c, max_seq, 40, page, seqs, max_tokens, prefix, norm, kv_dtype=dtype) as bp:
        try:
            at = 0
            for part in parts:
                n = len(part[0][0])
                bp.prefixStep(at, n)
                for layer in range(c.block_count):
                    bp.forwardBatch(layer, *upload(d, c, part[layer], max_tokens))
                at += n
            lengths = np.full(seqs, prefix, I)
            bp.setLengths(lengths)
            for i, grow in enumerate(steps):
                print(f"[gpu] {name} cache {dtype} step {i}", flush=True)
                n = sum(max(g, 0) for g in grow)
                rows = step_inputs(rng, c, n)
                bp.setGrow(np.array(grow, I))
                bp.step()
                assert bp.status() == 0
                starts = np.concatenate([[0], np.cumsum(np.maximum(grow, 0))])
                outs = []
                for layer in range(c.block_count):
                    bp.gpuXb2.upload(np.full(max_tokens * c.q_dim, 77, F32))
                    bp.forwardBatch(layer, *upload(d, c, rows[layer], max_tokens))
                    outs.append(bp.downloadOut())
                    assert (outs[layer][n:] == 77).all()
                for b, g in enumerate(grow):
                    if g > 0:
                        mine = [[x[starts[b]:starts[b + 1]] for x in r] for r in rows]
                        want = singles[b].step(mine)
                        for layer in range(c.block_count):
                            err = np.abs(outs[layer][starts[b]:starts[b + 1]] - want[layer]).max()
                            assert err < 2e-5, (i, b, layer, err)   # both are within 1e-5 of 64 bits
                    lengths[b] = 0 if g < 0 else lengths[b] + g
                assert np.array_equal(bp.lengths(), lengths)
                for b, g in enumerate(grow):
                    if g < 0:    # the row begins again behind the prefix
                        lengths[b] = prefix
                        singles[b].fp.close()
                        singles[b] = Single(c, max_seq, norm, dtype, parts)
                bp.setLengths(lengths)
        finally:
            for s in singles:
                s.fp.close()


def test_captured_step_replays_as_sequences_grow():
    """Tables, append and attention of two layers in one graph: every replay equals the eager steps of
    a second pass bit for bit, with eager work of that pass between the replays."""
    c = CONFIGS["llama"]
    rng = np.random.default_rng(2)
    max_seq, page, prefix, seqs, max_tokens = 200, 16, 32, 6, 12
    part = step_inputs(rng, c, 32)
    grows = [rng.integers(0, 3, seqs).astype(I) for _ in range(8)]
    with pc.Device() as d, HipBatchPass(c, max_seq, 90, page, seqs, 40, prefix) as a, \
            HipBatchPass(c, max_seq, 90, page, seqs, 40, prefix) as b:
        bufs = [[d.up(np.zeros((40, w), F32)) for w in (c.q_dim, c.kv_dim, c.kv_dim)] for _ in range(c.block_count)]
        outs = {x: [d.up(np.zeros((40, c.q_dim), F32)) for _ in range(c.block_count)] for x in (a, b)}

        def put(rows):
            for layer in range(c.block_count):
                for p, x in zip(bufs[layer], rows[layer]):
                    x = np.ascontiguousarray(x)
                    _lib.call("llmp_memcpy_htod", p, x.ctypes.data, x.nbytes, 0)

        def step(x):
            x.step()
            for layer in range(c.block_count):
                x.forwardBatch(layer, *bufs[layer])
                _lib.call("llmp_memcpy_dtod", outs[x][layer], x.gpuXb2.ptr, 40 * c.q_dim * 4, 0)
        put(part)
        for x in (a, b):
            x.prefixStep(0, 32)
            for layer in range(c.block_count):
                x.forwardBatch(layer, *bufs[layer])
            x.setLengths(np.full(seqs, prefix, I))
        # one eager step of both, which also sizes the workspaces
        put(step_inputs(rng, c, 40))
        for x in (a, b):
            x.setGrow(grows[0])
            step(x)
        g = C.c_uint64()
        _lib.call("llmp_graph_begin", 0)
        step(a)
        _lib.call("llmp_graph_end", 0, C.byref(g))
        for i, grow in enumerate(grows[1:]):
            print(f"[gpu] replay {i}", flush=True)
            put(step_inputs(rng, c, 40))
            for x in (a, b):
                x.setGrow(grow)
            _lib.call("llmp_graph_launch", g.value, 0)
            step(b)
            _lib.call("llmp_stream_sync", 0)
            n = int(grow.sum())
            assert a.status() == 0 and np.array_equal(a.lengths(), b.lengths())
            for layer in range(c.block_count):
                x, y = (d.down(outs[z][layer], F32, (40, c.q_dim))[:n] for z in (a, b))
                assert np.array_equal(x.view(np.uint32), y.view(np.uint32)), (i, layer)
                p, r = a.kv.read(layer), b.kv.read(layer)
                used = np.zeros((90, page), bool)
                blocks, lengths = a.gpuBlocks.download(I).reshape(seqs, -1), a.lengths()
                for s in range(seqs):
                    j = np.arange(lengths[s])
                    used[blocks[s][j // page], j % page] = True
                for w in p:
                    assert np.array_equal(p[w].transpose(0, 2, 1, 3)[used], r[w].transpose(0, 2, 1, 3)[used]), (i, layer, w)
        _lib.call("llmp_graph_destroy", g.value)


def test_a_captured_call_does_not_grow_its_workspace():
    c = CONFIGS["llama"]
    with pc.Device() as d, HipBatchPass(c, 64, 8, 16, 2, 4) as a:
        bufs = [d.up(np.zeros((4, w), F32)) for w in (c.q_dim, c.kv_dim, c.kv_dim)]
        a.setGrow(np.array([1, 1], I))
        a.step()
        g = C.c_uint64()
        _lib.call("llmp_graph_begin", 0)
        with pytest.raises(_lib.LlmpError) as e:
            a.forwardBatch(0, *bufs)
        assert e.value.code == 1 and "captured" in str(e.value)
        _lib.call("llmp_graph_end", 0, C.byref(g))
        _lib.call("llmp_graph_destroy", g.value)
        a.forwardBatch(0, *bufs)
        a.sync()
