"""The operators of a batch of sequences over one paged KV pool, as cases to time and to compare:
what each listed case stands for is said beside it in `listed`.

  tables   block tables, positions and slots of one step, from the lengths of the requests
           (llmp_paged_tables);
  append   rotation of the queries and keys of a ragged batch of tokens, and the K and V rows
           stored at their slots (llmp_paged_append);
  attn     attention of those tokens: a prefix that every sequence shares is read once for all of
           them, each sequence's own rows through its block table (llmp_paged_attn).

A pool holds pages of `page` rows per KV head: K [pages][heads][page][d] and V the same, fp32, or
int8 quants with one fp32 scale per 32 values.  With `own` the library's entry points run, on a
stream of their own; without it `run` is the same mathematics in elementary operations."""
import ctypes
import math
import random

import torch

own = False
DEV = "cuda:0"
EPS = 1e-6
# query heads, KV heads, head_dim, QK-norm, half layout of the rotated pairs, window
SHAPES = {
    "32/8/64": (32, 8, 64, False, False, 0),
    "32/8/128": (32, 8, 128, False, False, 0),
    "16/8/128": (16, 8, 128, True, True, 0),
    "24/8/96": (24, 8, 96, False, True, 0),
    "4/1/256": (4, 1, 256, True, False, 512),
}
THETA = 1e6


def _attn(shape, page, prefix, batch, held, new, cache="f32", lengths=1):
    """`held`: the most rows of its own that a sequence has before its new tokens; `new`: the most
    new tokens (1: one each)."""
    return {"kind": "attn", "shape": shape, "page": page, "prefix": prefix, "batch": batch, "held": held,
            "new": new, "cache": cache, "lengths": lengths}


def _append(shape, page, tokens, far, part=1.0, scaled=1.0, inputs="f32", merged=False, cache="f32", lengths=1):
    """`far`: positions go up to here; `part`: the rotated part of a head; `scaled`: the factor by
    which the table stretches the trained context; `merged`: q, k and v are parts of one row."""
    return {"kind": "append", "shape": shape, "page": page, "tokens": tokens, "far": far, "part": part,
            "scaled": scaled, "inputs": inputs, "merged": merged, "cache": cache, "lengths": lengths}


def _tables(page, seqs, held, new, done, shared, lengths=1):
    """`held`: the longest sequence; `new`: the most new tokens of one; `done`: the share of
    sequences that have ended; `shared`: the blocks of the common prefix."""
    return {"kind": "tables", "page": page, "seqs": seqs, "held": held, "new": new, "done": done,
            "shared": shared, "lengths": lengths}


def listed():
    def c(name, f, *a, **k):
        return dict(f(*a, **k), name=name)
    return [
        # Two samples of a short prompt with a small model: launches and latency are all there is.
        c("attn_two_samples", _attn, "32/8/64", 16, 173, 2, 30, 1),
        # Sixteen samples of one prompt, some hundred tokens in.
        c("attn_samples", _attn, "16/8/128", 16, 4001, 16, 300, 1),
        # Many chats under one system prompt, over the 8-bit cache that many sequences need.
        c("attn_chats_q8", _attn, "32/8/64", 32, 6144, 64, 2000, 1, cache="q8_0"),
        # Questions about one long document, asked together.
        c("attn_document", _attn, "32/8/128", 64, 32001, 32, 1500, 1),
        # Draft tokens of twelve sequences to verify, windowed layer of one KV head.
        c("attn_drafts_window", _attn, "4/1/256", 16, 300, 12, 900, 9),
        # Twelve new chats whose first turns are computed after the system prompt.
        c("attn_turns", _attn, "32/8/64", 16, 2000, 12, 0, 700),
        # One decode step of 32 sequences, with QK-norm and halves.
        c("append_step", _append, "16/8/128", 16, 32, 8191),
        # The prompts of one step in bf16 from a merged projection, rotary positions stretched
        # eightfold.
        c("append_prompts", _append, "32/8/128", 64, 4099, 32767, scaled=8.0, inputs="bf16", merged=True),
        # The same over the 8-bit cache, half of each head rotated.
        c("append_q8", _append, "32/8/64", 32, 1500, 16383, part=0.5, cache="q8_0"),
        # The tables of one decode step.
        c("tables_step", _tables, 16, 48, 4000, 1, 0.05, 100),
        # A step that ends some sequences and takes in new prompts.
        c("tables_prompts", _tables, 16, 300, 3000, 900, 0.2, 8),
        # A large service: thousands of sequences, a few tokens each.
        c("tables_service", _tables, 64, 4096, 8000, 4, 0.1, 3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "append", "tables"))
    lengths, page = rng.randint(2, 1 << 20), rng.choice((16, 32, 64, 128))
    if kind == "tables":
        seqs = _log(rng, 1, 4096)
        new = rng.choice((1, _log(rng, 2, max(2, min(2000, 60000 // seqs)))))
        return _tables(page, seqs, _log(rng, 4 * page, 8000), new, rng.choice((0.0, 0.1, 0.4)), rng.randint(0, 3), lengths)
    shape = rng.choice(sorted(SHAPES))
    d, norm = SHAPES[shape][2], SHAPES[shape][3]
    if kind == "append":
        cache = "q8_0" if not norm and d != 96 and rng.random() < 0.4 else "f32"
        return _append(shape, page, _log(rng, 1, 4099), _log(rng, 4100, 32767), rng.choice((1.0, 1.0, 0.5, 0.25)),
                       rng.choice((1.0, 1.0, 4.0, 8.0)), rng.choice(("f32", "bf16")), rng.random() < 0.5, cache, lengths)
    cache = "q8_0" if d != 96 and rng.random() < 0.4 else "f32"
    c = _attn(shape, page, rng.choice((0, _log(rng, 17, 32000), _log(rng, 17, 32000))), _log(rng, 1, 64),
              _log(rng, 1, 2000), rng.choice((1, 1, 1, rng.randint(2, 17), _log(rng, 18, 700))), cache, lengths)
    while work(c)["flops"] > 7e10 or work(c)["bytes"] > 6e8:
        c.update(batch=max(1, c["batch"] * 2 // 3), prefix=c["prefix"] * 3 // 4, held=c["held"] * 3 // 4 + 1)
    return c


# ------------------------------------------------------------------------- sizes of a case
def _lengths(case):
    """Rows held and new tokens of each sequence."""
    rng = random.Random(case["lengths"])
    if case["kind"] == "attn":
        held = [case["prefix"] + rng.randint(case["held"] // 20, max(case["held"], 1)) for _ in range(case["batch"])]
        if case["held"] == 0:
            held = [case["prefix"]] * case["batch"]
        new = [rng.randint(1 + case["new"] // 20, max(1, case["new"])) for _ in range(case["batch"])]
        return held, new
    low = case["shared"] * case["page"]
    held, grow = [], []
    for _ in range(case["seqs"]):
        first = rng.random() < (0.4 if case["new"] > 8 else 0.02)
        held.append(low if first else max(low, _log(rng, case["page"], max(case["held"], case["page"] + 1))))
        grow.append(-1 if not first and rng.random() < case["done"] else rng.randint(case["new"] // 9, case["new"]))
    return held, grow


def _seen(case, p):
    """Rows that a token at position p attends, and where they begin."""
    w = SHAPES[case["shape"]][5]
    start = max(0, p + 1 - w) if w else 0
    return p + 1 - start, start


def _up(a, b):
    return -(-a // b)


def work(case):
    if case["kind"] == "tables":
        held, grow = _lengths(case)
        p, tokens = case["page"], sum(max(g, 0) for g in grow)
        pages = sum(_up(h + g, p) - _up(h, p) if g >= 0 else max(0, _up(h, p) - case["shared"]) for h, g in zip(held, grow))
        return {"bytes": 16.0 * case["seqs"] + 8.0 * pages + 12.0 * tokens, "flops": 0.0}
    hq, hkv, d = SHAPES[case["shape"]][:3]
    row = d * 4 if case["cache"] == "f32" else d + d // 8
    if case["kind"] == "append":
        t, size = case["tokens"], 4 if case["inputs"] == "f32" else 2
        turned = int(d * case["part"]) // 2
        return {"bytes": t * (size * (hq + 2 * hkv) * d + 4.0 * hq * d + 2 * hkv * row + 8 * turned + 8),
                "flops": 6.0 * t * (hq + hkv) * turned}
    held, new = _lengths(case)
    tokens, low, rows, seen = sum(new), case["prefix"], 0, 0
    for h, n in zip(held, new):
        start = _seen(case, h)[1]
        low = min(low, start)
        rows += h + n - max(start, case["prefix"])
        seen += sum(_seen(case, p)[0] for p in range(h, h + n))
    return {"bytes": 2.0 * hkv * row * (rows + case["prefix"] - low) + 8.0 * tokens * hq * d, "flops": 4.0 * hq * d * seen}


# ------------------------------------------------------------------------------- the state
class _State:
    pass


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _pad(n):
    return (n + 255) // 256 * 256


def _pool(case, pages, g=None):
    """The pool's memory, as the library divides it, and its planes; filled where `g` is given."""
    hkv, d, page = SHAPES[case["shape"]][1], SHAPES[case["shape"]][2], case["page"]
    n = pages * hkv * page * d
    q8 = case["cache"] != "f32"
    plane, scale = _pad(n if q8 else 4 * n), _pad(n // 8) if q8 else 0
    mem = torch.zeros(2 * (plane + scale), dtype=torch.uint8, device=DEV)
    shape, at, planes = (pages, hkv, page, d), 0, {}
    for w in ("k", "v"):
        t = mem[at:at + (n if q8 else 4 * n)].view(torch.int8 if q8 else torch.float32).view(shape)
        at += plane
        planes[w] = t
        if q8:
            s = mem[at:at + n // 8].view(torch.float32).view(pages, hkv, page, d // 32)
            at += scale
            planes[w + "s"] = s
        if g is not None:
            # K is scaled so that the scores spread over a few units, as a trained model's do.
            size = 2.0 if w == "k" else 1.0
            if q8:
                t.copy_(torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8))
                s.copy_((torch.rand(s.shape, generator=g, device=DEV) + 0.5) * (size / 73))
            else:
                t.normal_(generator=g).mul_(size)
    return mem, planes


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _turns(case, rows):
    """Angles [rows][pairs] of the positions, in 64 bits.  Stretched contexts: the frequencies that
    turn less than once over the trained length are divided by the factor, those that turn more than
    32 times are kept, and those between are blended linearly in the index."""
    d = SHAPES[case["shape"]][2]
    r = int(d * case["part"])
    i = torch.arange(r // 2, device=DEV, dtype=torch.float64)
    f = THETA ** (-2 * i / r)
    if case["scaled"] > 1:
        trained = 4096

        def index(turns):
            return r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(THETA))
        lo, hi = max(0, math.floor(index(32))), min(r - 1, math.ceil(index(1)))
        keep = 1 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f / case["scaled"] * (1 - keep) + f * keep
    return torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * f


def _gammas(d):
    """Weights of the per-head norms: the model's, alike for every input."""
    i = torch.arange(d, device=DEV, dtype=torch.float32)
    return 1 + 0.25 * torch.cos(0.37 * i), 1 + 0.25 * torch.sin(0.53 * i)


def prepare(case, seed):
    g, s = _generator(seed), _State()
    s.case, s.seed, s.page = case, seed, case["page"]
    rng = random.Random(case["lengths"] + 1)
    if case["kind"] == "tables":
        held, grow = _lengths(case)
        s.n, p = case["seqs"], case["page"]
        s.most = max(h + max(x, 0) for h, x in zip(held, grow))
        s.width = _up(s.most, p)
        shared = list(range(case["shared"]))
        need = sum(_up(h + max(x, 0), p) for h, x in zip(held, grow))
        s.pages = case["shared"] + need + 64
        order = torch.randperm(s.pages - case["shared"], generator=g, device=DEV, dtype=torch.int32) + case["shared"]
        have = _ints([_up(h, p) for h in held])[:, None]
        j = torch.arange(s.width, device=DEV, dtype=torch.int32)[None]
        mine = (j >= case["shared"]) & (j < have)
        s.blocks = torch.full((s.n, s.width), -1, dtype=torch.int32, device=DEV)
        s.blocks[:, :len(shared)] = _ints(shared)
        used = int(mine.sum())
        s.blocks[mine] = order[:used]
        s.free = torch.full((s.pages,), -1, dtype=torch.int32, device=DEV)
        s.free[:s.pages - case["shared"] - used] = order[used:]
        s.n_free = _ints([s.pages - case["shared"] - used])
        s.len, s.grow = _ints(held), _ints(grow)
        s.tokens = sum(max(x, 0) for x in grow) + 5
        s.len_out, s.n_free_out, s.status = torch.empty_like(s.len), torch.empty_like(s.n_free), _ints([-9])
        s.seq_start = torch.empty(s.n + 1, dtype=torch.int32, device=DEV)
        s.positions, s.slots = (torch.empty(s.tokens, dtype=torch.int32, device=DEV) for _ in range(2))
        return s
    hq, hkv, d, norm, half, window = SHAPES[case["shape"]]

    def normal(*size):
        return torch.randn(size, generator=g, device=DEV)
    if case["kind"] == "append":
        t, p = case["tokens"], case["page"]
        s.pages = _up(t, p) + 3
        s.mem, s.planes = _pool(case, s.pages)
        s.positions = torch.randint(0, case["far"] + 1, (t,), generator=g, device=DEV, dtype=torch.int32)
        s.slots = torch.randperm(s.pages * p, generator=g, device=DEV, dtype=torch.int32)[:t].contiguous()
        a = _turns(case, case["far"] + 1)
        s.cos, s.sin = torch.cos(a).float(), torch.sin(a).float()
        s.gammas = _gammas(d) if norm else None
        dt = torch.float32 if case["inputs"] == "f32" else torch.bfloat16
        rows = normal(t, (hq + 2 * hkv) * d).to(dt)
        s.parts = rows.split((hq * d, hkv * d, hkv * d), 1)
        if not case["merged"]:
            s.parts = tuple(x.contiguous() for x in s.parts)
        s.out = torch.empty((t, hq, d), device=DEV)
        s.most = case["far"] + 1
        return s
    held, new = _lengths(case)
    p, s.n = case["page"], case["batch"]
    s.most = max(h + n for h, n in zip(held, new))
    s.width = _up(s.most, p)
    # The last block of the prefix is every sequence's own where the prefix ends inside it.
    whole = case["prefix"] // p
    s.pages = _up(case["prefix"], p) + sum(_up(h + n, p) - whole for h, n in zip(held, new)) + 2
    s.mem, s.planes = _pool(case, s.pages, g)
    order = torch.randperm(s.pages, generator=g, device=DEV, dtype=torch.int32)
    s.blocks = torch.full((s.n, s.width), -1, dtype=torch.int32, device=DEV)
    s.blocks[:, :whole] = order[:whole]
    at = whole
    have = _ints([_up(h + n, p) for h, n in zip(held, new)])[:, None]
    j = torch.arange(s.width, device=DEV, dtype=torch.int32)[None]
    mine = (j >= whole) & (j < have)
    s.blocks[mine] = order[at:at + int(mine.sum())]
    s.seq_start = _ints([0] + torch.tensor(new).cumsum(0).tolist())
    s.positions = _ints([h + i for h, n in zip(held, new) for i in range(n)])
    s.tokens, s.prefix, s.longest_new = sum(new), case["prefix"], max(new)
    s.q = normal(s.tokens, hq, d)
    s.out = torch.empty((s.tokens, hq, d), device=DEV)
    return s


# ------------------------------------------------------------------------------- the library
_kept = {}


def _lib():
    from llmplayer_amd import _lib as lib
    if "stream" not in _kept:
        lib.call("llmp_init", 0)
        _kept["stream"] = torch.cuda.Stream()
    return lib, _kept["stream"].cuda_stream


def _handle(s):
    """The handle that a program keeps for its model and pool geometry."""
    lib, _ = _lib()
    case = s.case
    hq, hkv, d, norm, half, window = SHAPES[case.get("shape", "32/8/64")]
    part, scaled = case.get("part", 1.0), case.get("scaled", 1.0)
    cache = lib.LLMP_KV_F32 if case.get("cache", "f32") == "f32" else lib.LLMP_KV_Q8_0
    key = (case["kind"], case.get("shape"), s.page, s.pages, s.most, cache, part, scaled)
    if key not in _kept:
        h = ctypes.c_uint64()
        lib.call("llmp_paged_create", 1, s.pages, s.page, s.most, hkv, d, cache, ctypes.byref(h))
        if case["kind"] == "append":
            fp = ctypes.POINTER(ctypes.c_float)
            tables = [x.cpu() for x in (s.cos, s.sin)]
            lib.call("llmp_rope_upload", h.value, lib.LLMP_ROPE_SEL_GLOBAL, *(ctypes.cast(x.data_ptr(), fp) for x in tables),
                     s.most, s.cos.shape[1])
            w = [x.cpu() for x in s.gammas] if norm else None
            qn, kn = (ctypes.cast(x.data_ptr(), fp) for x in w) if norm else (None, None)
            lib.call("llmp_layer_config", h.value, 0, hq, hkv, d, lib.LLMP_ROPE_NEOX if half else lib.LLMP_ROPE_NORMAL,
                     lib.LLMP_ROPE_SEL_GLOBAL, 0, 1, 0.0, 0.0, EPS, qn, kn)
        elif case["kind"] == "attn":
            lib.call("llmp_layer_config", h.value, 0, hq, hkv, d, lib.LLMP_ROPE_NORMAL, lib.LLMP_ROPE_SEL_NONE, window, 0,
                     0.0, 0.0, EPS, None, None)
        _kept[key] = h.value
    return _kept[key]


def _run_own(s):
    lib, st = _lib()
    h, case = _handle(s), s.case
    if case["kind"] == "tables":
        lib.call("llmp_paged_tables", h, s.n, case["shared"], s.tokens, s.len.data_ptr(), s.grow.data_ptr(),
                 s.free.data_ptr(), s.n_free.data_ptr(), s.blocks.data_ptr(), s.len_out.data_ptr(),
                 s.n_free_out.data_ptr(), s.seq_start.data_ptr(), s.positions.data_ptr(), s.slots.data_ptr(),
                 s.status.data_ptr(), st)
        return _tables_out(s)
    lib.call("llmp_paged_bind", h, s.mem.data_ptr())
    if case["kind"] == "append":
        q, k, v = s.parts
        lib.call("llmp_paged_append", h, 0, case["tokens"], s.positions.data_ptr(), s.slots.data_ptr(),
                 lib.LLMP_IN_F32 if case["inputs"] == "f32" else lib.LLMP_IN_BF16, q.data_ptr(), q.stride(0),
                 k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), s.out.data_ptr(), s.out.stride(0), st)
        with torch.cuda.stream(_kept["stream"]):
            return _append_out(s)
    hq, d = SHAPES[case["shape"]][0], SHAPES[case["shape"]][2]
    lib.call("llmp_paged_attn", h, 0, s.n, s.tokens, s.prefix, s.most, s.seq_start.data_ptr(), s.positions.data_ptr(),
             s.blocks.data_ptr(), s.q.data_ptr(), hq * d, 0, s.out.data_ptr(), hq * d, st)
    return s.out


def _tables_out(s):
    return {"blocks": s.blocks, "len": s.len_out, "n_free": s.n_free_out, "free": s.free, "seq_start": s.seq_start,
            "positions": s.positions, "slots": s.slots, "status": s.status}


def _append_out(s):
    """The rotated queries and the pool; int8 rows as the values that they stand for."""
    p = s.planes
    if s.case["cache"] == "f32":
        return {"q": s.out, "k": p["k"], "v": p["v"]}
    k, v = (p[w].view(p[w + "s"].shape + (32,)) * p[w + "s"][..., None] for w in ("k", "v"))
    return {"q": s.out, "k": k, "v": v}


# ------------------------------------------------------------------------------ plain forms
def _run_tables(s):
    p, shared = s.page, s.case["shared"]
    done = s.grow < 0
    new = s.grow.clamp(min=0)
    have = torch.div(s.len + p - 1, p, rounding_mode="floor")
    after = torch.div(s.len + new + p - 1, p, rounding_mode="floor")
    need = torch.where(done, 0, after - have)
    back = torch.where(done, (have - shared).clamp(min=0), 0)
    short = need.sum() - back.sum() - s.n_free[0]
    over = ((s.len < 0) | (s.len + new > s.most)).any()
    many = new.sum() > s.tokens
    status = torch.where(over, -1, torch.where(many, -2, short.clamp(min=0))).int()
    good = status == 0
    new = new * good
    done = done & good
    j = torch.arange(s.width, device=DEV, dtype=torch.int32)[None]
    returned = done[:, None] & (j >= shared) & (j < have[:, None])
    taken = (good & ~done)[:, None] & (j >= have[:, None]) & (j < after[:, None])
    top = s.n_free[0] + returned.sum()
    s.free[(s.n_free[0] + torch.cumsum(returned.flatten(), 0) - 1)[returned.flatten()]] = s.blocks[returned]
    s.blocks[taken] = s.free[(top - torch.cumsum(taken.flatten(), 0))[taken.flatten()]]
    s.len_out.copy_(torch.where(done, 0, s.len + new))
    s.n_free_out.copy_((top - taken.sum())[None])
    ends = torch.cumsum(new, 0)
    s.seq_start.copy_(torch.cat([ends.new_zeros(1), ends]))
    i = torch.arange(s.tokens, device=DEV)
    real = i < ends[-1]
    b = torch.searchsorted(ends, i, right=True).clamp(max=s.n - 1)
    at = (s.len[b] + i - (ends - new)[b]).clamp(min=0, max=s.width * p - 1)
    page = s.blocks[b, torch.div(at, p, rounding_mode="floor")]
    s.positions.copy_(torch.where(real, at, -1))
    s.slots.copy_(torch.where(real, page * p + at % p, -1))
    s.status.copy_(status[None])
    return _tables_out(s)


def _rotated(x, c, sn, half, norm):
    """x [t][heads][d] in 32 bits; c, sn [t][pairs]."""
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
    n = c.shape[1]
    c, sn, turn, rest = c[:, None], sn[:, None], x[..., :2 * n], x[..., 2 * n:]
    if half:
        a, b = turn[..., :n], turn[..., n:]
        return torch.cat([a * c - b * sn, a * sn + b * c, rest], -1)
    a, b = turn[..., 0::2], turn[..., 1::2]
    return torch.cat([torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2), rest], -1)


def _run_append(s):
    hq, hkv, d, norm, half, _ = SHAPES[s.case["shape"]]
    at, slot = s.positions.long(), s.slots.long()
    c, sn = s.cos[at], s.sin[at]
    q, k, v = (x.float().reshape(x.shape[0], -1, d) for x in s.parts)
    gq, gk = s.gammas if norm else (None, None)
    s.out.copy_(_rotated(q, c, sn, half, gq))
    rows = {"k": _rotated(k, c, sn, half, gk), "v": v}
    page, row = torch.div(slot, s.page, rounding_mode="floor"), slot % s.page
    for w, x in rows.items():
        if s.case["cache"] == "f32":
            s.planes[w][page, :, row] = x
            continue
        b = x.reshape(x.shape[0], hkv, d // 32, 32)
        scale = b.abs().amax(-1) / 127
        codes = b * torch.where(scale > 0, 1 / scale, 0)[..., None]
        codes = torch.where(codes - codes.floor() >= 0.5, codes.floor() + 1, codes.floor()).clamp(-128, 127)
        s.planes[w][page, :, row] = codes.reshape(x.shape).to(torch.int8)
        s.planes[w + "s"][page, :, row] = scale
    return _append_out(s)


def _rows(s, w, page, row, dtype):
    """Rows of the pool [...][heads][d]."""
    x = s.planes[w][page, :, row].to(dtype)
    if s.case["cache"] != "f32":
        x = (x.view(x.shape[:-1] + (-1, 32)) * s.planes[w + "s"][page, :, row].to(dtype)[..., None]).flatten(-2)
    return x


def _part(q, k, v, hide):
    """Largest score, sum and unnormalised output of the queries q [n][m][d] over k, v [n][rows][d]."""
    sc = torch.bmm(q, k.transpose(1, 2).contiguous())
    sc.masked_fill_(hide, -math.inf)
    m = sc.amax(-1, keepdim=True).clamp(min=-1e30)
    e = sc.sub_(m).exp_()
    return m, e.sum(-1, keepdim=True), torch.bmm(e, v)


def _run_attn(s):
    hq, hkv, d, _, _, window = SHAPES[s.case["shape"]]
    grp, t, b, p = hq // hkv, s.tokens, s.n, s.page
    at = s.positions.long()
    q = (s.q / math.sqrt(d)).view(t, hkv, grp, d)
    parts = []
    if s.prefix:
        j = torch.arange(s.prefix, device=DEV)
        page, row = s.blocks[0].long()[torch.div(j, p, rounding_mode="floor")], j % p
        k, v = (_rows(s, w, page, row, torch.float32).transpose(0, 1).contiguous() for w in ("k", "v"))
        hide = j[None] > at[:, None]
        if window:
            hide |= j[None] <= at[:, None] - window
        hide = hide[:, None].expand(t, grp, s.prefix).reshape(1, t * grp, s.prefix)
        x = _part(q.transpose(0, 1).reshape(hkv, t * grp, d).contiguous(), k, v, hide)
        parts.append([y.view(hkv, t, grp, -1).transpose(0, 1) for y in x])
    # Each sequence's own rows, padded to the longest; its queries padded to the most of one.
    first, size = s.seq_start[:-1].long(), (s.seq_start[1:] - s.seq_start[:-1]).long()
    i = torch.arange(s.longest_new, device=DEV)
    token = (first[:, None] + i).clamp(max=t - 1)
    real = i[None] < size[:, None]
    qp = q[token].permute(0, 2, 1, 3, 4).reshape(b * hkv, s.longest_new * grp, d).contiguous()
    j = torch.arange(s.prefix, s.most, device=DEV)
    page = s.blocks.long()[:, torch.div(j, p, rounding_mode="floor")].clamp(min=0)
    k, v = (_rows(s, w, page, (j % p).expand(b, -1), torch.float32).transpose(1, 2).reshape(b * hkv, len(j), d) for w in ("k", "v"))
    pos = at[token]
    hide = j > pos[..., None]
    if window:
        hide |= j <= pos[..., None] - window
    hide = hide[:, None, :, None].expand(b, hkv, s.longest_new, grp, len(j)).reshape(b * hkv, -1, len(j))
    x = _part(qp, k, v, hide)
    parts.append([y.view(b, hkv, s.longest_new, grp, -1).transpose(1, 2)[real] for y in x])
    m = torch.stack([y[0] for y in parts]).amax(0)
    f = [torch.exp(y[0] - m) for y in parts]
    total = sum(y[1] * w for y, w in zip(parts, f))
    s.out.copy_((sum(y[2] * w for y, w in zip(parts, f)) / total).reshape(t, hq, d))
    return s.out


def run(s):
    if own:
        return _run_own(s)
    return {"tables": _run_tables, "append": _run_append, "attn": _run_attn}[s.case["kind"]](s)


# ---------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    hq, hkv, d, norm, half, window = SHAPES[case["shape"]]
    if case["kind"] == "append":
        a = _turns(case, case["far"] + 1)[s.positions.long()]
        turn = torch.polar(torch.ones_like(a), a)[:, None]

        def rotate(x, w):
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
            n = a.shape[1]
            i = torch.arange(n, device=DEV)
            one, two = (i, i + n) if half else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., one], x[..., two]) * turn
            x = x.clone()
            x[..., one], x[..., two] = z.real, z.imag
            return x
        q, k, v = (x.double().reshape(case["tokens"], -1, d) for x in s.parts)
        got = {"q": rotate(q, s.gammas[0] if norm else None), "k": None, "v": None}
        if case["cache"] == "f32":
            for w, x in (("k", rotate(k, s.gammas[1] if norm else None)), ("v", v)):
                got[w] = torch.zeros((s.pages * case["page"], hkv, d), dtype=torch.float64, device=DEV)
                got[w][s.slots.long()] = x
                got[w] = got[w].view(s.pages, case["page"], hkv, d).transpose(1, 2).contiguous()
        return got
    held, new = _lengths(case)
    out = torch.empty((s.tokens, hq, d), dtype=torch.float64, device=DEV)
    at = 0
    for b, (h, n) in enumerate(zip(held, new)):
        rows = torch.arange(h + n, device=DEV)
        entry = torch.where(rows < case["prefix"], s.blocks[0].long()[rows // case["page"]], s.blocks[b].long()[rows // case["page"]])
        k, v = (_rows(s, w, entry, rows % case["page"], torch.float64) for w in ("k", "v"))
        pos = torch.arange(h, h + n, device=DEV)[:, None]
        hide = (rows[None] > pos) | ((rows[None] <= pos - window) if window else (rows[None] < 0))
        for head in range(hq):
            kv = head // (hq // hkv)
            sc = (s.q[at:at + n, head].double() @ k[:, kv].t()) / math.sqrt(d)
            out[at:at + n, head] = torch.softmax(sc.masked_fill(hide, -math.inf), -1) @ v[:, kv]
        at += n
    return out
