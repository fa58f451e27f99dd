"""Operators of a paged key/value cache: what a program that serves several sequences has the library do.

``rotate`` norms the heads of queries and keys and rotates them by their positions; ``append``
stores new keys (normed and rotated on the way) and values in a cache of pages, as 16-bit floats or
as 4-bit codes, and reads them back; ``read`` restores cached rows; ``attend`` is attention of
each sequence's last rows over its pages, for single tokens, drafted tokens and prompts.  Head
shapes are those of ``brisk_hip.synth.SPECS``.  Inputs are random, made from the seed on the GPU.

A 4-bit row holds blocks of 32 values: a scale d, the block's first value of largest magnitude
divided by -8 and rounded to 16 bits, and a code n = floor(x / d + 8.5), at most 15, for each value;
it stands for (n - 8) d.
"""
import ctypes as C
import math
import random
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
GGML = {"f32": 0, "f16": 1, "bf16": 30, "q4_0": 2}  # the library's type numbers
BASE = 1e6      # the rotation's base
EPS = 1e-6
CHUNK = 32      # values that share a scale


def listed():
    return [
        # one new token's queries and keys, normed and rotated: launch and latency
        {"name": "rotate_token", "kind": "rotate", "n": 1, "heads": 16, "kv_heads": 8, "head_dim": 128, "rotated": 128, "half": True,
         "norm": True, "input": "f32", "output": "f16", "context": 40960},
        # a long prompt's, adjacent pairs, no norms
        {"name": "rotate_prompt", "kind": "rotate", "n": 4011, "heads": 32, "kv_heads": 8, "head_dim": 64, "rotated": 64, "half": False,
         "norm": False, "input": "f32", "output": "bf16", "context": 131072},
        # the decode step of 48 sequences, into 4 bits
        {"name": "append_tokens_q4", "kind": "append", "seqs": 48, "rows": 1, "length": 3000, "heads": 16, "kv_heads": 8, "head_dim": 128,
         "rotated": 128, "half": True, "norm": True, "input": "f32", "cache": "q4_0", "page": 16},
        # prompts of several sequences, of unequal length, a quarter of each head rotated, into 16 bits
        {"name": "append_prompts_f16", "kind": "append", "seqs": 5, "rows": 700, "length": 1900, "heads": 8, "kv_heads": 2, "head_dim": 256,
         "rotated": 64, "half": True, "norm": True, "input": "bf16", "cache": "f16", "page": 64},
        # a long prompt, into 4 bits
        {"name": "append_prompt_q4", "kind": "append", "seqs": 1, "rows": 8190, "length": 8190, "heads": 32, "kv_heads": 8, "head_dim": 64,
         "rotated": 64, "half": False, "norm": False, "input": "f32", "cache": "q4_0", "page": 32},
        # a short shared prefix restored for a session
        {"name": "read_prefix_f16", "kind": "read", "seqs": 1, "rows": 130, "length": 130, "kv_heads": 8, "head_dim": 128, "cache": "f16", "page": 16, "output": "f16"},
        # long conversations restored from 4 bits
        {"name": "read_long_q4", "kind": "read", "seqs": 4, "rows": 16000, "length": 16000, "kv_heads": 8, "head_dim": 128, "cache": "q4_0", "page": 64, "output": "f16"},
        # one sequence's next token early in a chat: latency
        {"name": "attend_token_short", "kind": "attend", "seqs": 1, "rows": 1, "length": 333, "heads": 16, "kv_heads": 8, "head_dim": 128,
         "window": 0, "input": "f16", "cache": "f16", "page": 16},
        # one sequence's next token late in a long document, held in 4 bits
        {"name": "attend_token_long_q4", "kind": "attend", "seqs": 1, "rows": 1, "length": 60001, "heads": 16, "kv_heads": 8, "head_dim": 128,
         "window": 0, "input": "f16", "cache": "q4_0", "page": 64},
        # the next tokens of 64 sequences of unequal length, held in 4 bits
        {"name": "attend_tokens_q4", "kind": "attend", "seqs": 64, "rows": 1, "length": 8000, "heads": 32, "kv_heads": 8, "head_dim": 64,
         "window": 0, "input": "bf16", "cache": "q4_0", "page": 16},
        # six drafted tokens of 8 sequences, wide heads behind a sliding window, 32-bit queries
        {"name": "attend_drafted_f32", "kind": "attend", "seqs": 8, "rows": 6, "length": 5000, "heads": 4, "kv_heads": 1, "head_dim": 256,
         "window": 512, "input": "f32", "cache": "f16", "page": 32},
        # the second part of a long prompt, held in 4 bits
        {"name": "attend_prompt_q4", "kind": "attend", "seqs": 1, "rows": 4000, "length": 8100, "heads": 16, "kv_heads": 8, "head_dim": 128,
         "window": 0, "input": "f16", "cache": "q4_0", "page": 64},
    ]


SHAPES = [(16, 8, 128), (32, 8, 64), (20, 5, 128), (4, 1, 256), (8, 2, 256), (16, 16, 96)]


def draw(rng):
    def between(lo, hi):  # over the logarithm
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["rotate", "append", "append", "read", "attend", "attend", "attend", "attend"])
    heads, kv_heads, dim = rng.choice(SHAPES)
    part = rng.choice([dim, dim, dim // 2, dim // 4])
    page = rng.choice([16, 32, 64, 128])
    cache = rng.choice(["q4_0", "q4_0", "f16"])
    turn = {"rotated": part, "half": rng.random() < 0.6, "norm": rng.random() < 0.5, "input": rng.choice(["f32", "f32", "bf16", "f16"])}
    if kind == "rotate":
        return {"kind": kind, "n": between(1, 4000), "heads": heads, "kv_heads": kv_heads, "head_dim": dim, **turn,
                "output": rng.choice(["f16", "bf16", "f32"]), "context": between(5000, 131072)}
    if kind == "append":
        seqs = between(1, 64)
        rows = 1 if rng.random() < 0.4 else between(2, 8000 // seqs)
        return {"kind": kind, "seqs": seqs, "rows": rows, "length": rows + between(1, 3000), "heads": heads, "kv_heads": kv_heads,
                "head_dim": dim, **turn, "cache": cache, "page": page}
    if kind == "read":
        seqs = between(1, 8)
        rows = between(1, 30000 // seqs)
        return {"kind": kind, "seqs": seqs, "rows": rows, "length": rows + between(1, 3000), "kv_heads": kv_heads, "head_dim": dim,
                "cache": cache, "page": page, "output": rng.choice(["f16", "f32", "bf16"])}
    sort = rng.choice(["token", "token", "drafted", "prompt"])
    if sort == "prompt":
        seqs = rng.choice([1, 1, 2, 3])
        rows = between(16, 4000 * 2048 // max(2048, heads * dim) // seqs)
        length = rows + between(1, 4000)
    else:
        seqs = between(1, 64)
        rows = 1 if sort == "token" else rng.randint(2, 8)
        length = rows + between(16, min(60000, 400000 // seqs))
    return {"kind": kind, "seqs": seqs, "rows": rows, "length": length, "heads": heads, "kv_heads": kv_heads, "head_dim": dim,
            "window": rng.choice([0, 0, 0, 512]), "input": rng.choice(["f16", "bf16", "f16", "f32"]), "cache": cache, "page": page}


# ---------------------------------------------------------------- inputs

def _batch(case):
    """(rows, lengths) of each sequence: the first has the case's own, the others fewer or as many."""
    r = random.Random("%(seqs)d/%(rows)d/%(length)d" % case)
    rows, lengths = [case["rows"]], [case["length"]]
    for _ in range(case["seqs"] - 1):
        rows.append(r.randint((case["rows"] + 1) // 2, case["rows"]))
        lengths.append(max(rows[-1], r.randint((case["length"] + 2) // 3, case["length"])))
    return rows, lengths


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(7919 * (int(seed) + 3))


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _keys(gen, n, heads, dim):
    """Keys as models have them: a few dimensions of each head are large."""
    return _normal(gen, n, heads, dim) * torch.exp(0.5 * _normal(gen, heads, dim))


def _table(positions, dims):
    """(cos, sin) pairs [positions, dims / 2, 2]; the angles in 64 bits, the later half of the positions' own scale as for a stretched context."""
    freq = BASE ** (-torch.arange(0, dims, 2, device="cuda", dtype=torch.float64) / dims)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq / 1.25
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    """The tensors of a case: rows as a fused projection leaves them, and what goes with them."""
    gen, kind, dim, kvh = _generator(seed), case["kind"], case["head_dim"], case["kv_heads"]
    d = {}
    if kind == "rotate":
        n, width = case["n"], (case["heads"] + 2 * kvh) * dim
        fused = (_normal(gen, n, width) * 1.5).to(TYPES[case["input"]])
        heads = fused.view(n, -1, dim)
        d["q"], d["k"] = heads[:, :case["heads"]], heads[:, case["heads"]:case["heads"] + kvh]
        d["positions"] = torch.randint(0, case["context"], (n,), device="cuda", generator=gen, dtype=torch.int32).sort()[0].int()
        d["table"] = _table(case["context"], case["rotated"])
        if case["norm"]:
            d["q_norm"], d["k_norm"] = 1 + 0.2 * _normal(gen, dim), 1 + 0.2 * _normal(gen, dim)
        return d
    rows, lengths = _batch(case)
    page, n = case["page"], sum(rows)
    counts = [-(-l // page) for l in lengths]
    d["pages"] = sum(counts) + 3
    order = torch.randperm(d["pages"], device="cuda", generator=gen).int()
    d["page_table"] = torch.zeros(len(rows), max(counts), dtype=torch.int32, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), torch.tensor(counts, device="cuda"))
    first = torch.tensor(np.cumsum([0] + counts[:-1]), device="cuda")
    at = torch.arange(sum(counts), device="cuda") - first[seq]
    d["page_table"][seq, at] = order[:sum(counts)]
    d["row_start"] = _ints([0] + list(np.cumsum(rows)))
    d["lengths"] = _ints(lengths)
    if kind == "append":
        width = (case["heads"] + 2 * kvh) * dim
        fused = _normal(gen, n, width)
        fused[:, case["heads"] * dim:(case["heads"] + kvh) * dim] = _keys(gen, n, kvh, dim).flatten(1)
        heads = fused.to(TYPES[case["input"]]).view(n, -1, dim)
        d["k"], d["v"] = heads[:, case["heads"]:case["heads"] + kvh], heads[:, case["heads"] + kvh:]
        d["table"] = _table(max(lengths), case["rotated"])
        if case["norm"]:
            d["k_norm"] = 1 + 0.2 * _normal(gen, dim)
        return d
    total = n if kind == "read" else sum(lengths)
    d["k"], d["v"] = _keys(gen, total, kvh, dim).half(), _normal(gen, total, kvh, dim).half()
    d["stored"] = d["row_start"] if kind == "read" else _ints([0] + list(np.cumsum(lengths)))
    if kind == "attend":
        d["q"] = (_normal(gen, n, case["heads"], dim) * 1.2).to(TYPES[case["input"]])
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    state = {"case": case, **d}
    if own:
        _prepare_own(state)
    elif case["kind"] != "rotate":
        state["where"] = _where(state["row_start"], state["lengths"], sum(_batch(case)[0]))
        shape = (d["pages"], case["page"], case["kv_heads"], case["head_dim"])
        state["cache"] = [_empty(case["cache"], shape), _empty(case["cache"], shape)]
        if case["kind"] != "append":
            seq, pos = _where(d["stored"], d["lengths"], d["k"].shape[0])
            for cache, x in zip(state["cache"], (d.pop("k"), d.pop("v"))):
                _store(case, cache, d["page_table"], seq, pos, x.double())
        state.pop("stored", None)
        if case["kind"] != "append":
            del state["k"], state["v"]
    return state


# ---------------------------------------------------------------- the plain forms

def _where(row_start, lengths, n):
    """Each row's sequence and position: a sequence's rows are its last ones."""
    seq = torch.searchsorted(row_start[1:].long().contiguous(), torch.arange(n, device="cuda"), right=True)
    pos = lengths.long()[seq] - row_start.long()[seq + 1] + torch.arange(n, device="cuda")
    return seq, pos


def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.to(x.dtype)


def _rotate(x, cs, half):
    """x [n, heads, dim], cs [n, rotated / 2, 2]."""
    r = 2 * cs.shape[1]
    c, s = cs[:, None, :, 0].to(x.dtype), cs[:, None, :, 1].to(x.dtype)
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if half else (x[..., 0:r:2], x[..., 1:r:2])
    a, b = a * c - b * s, a * s + b * c
    y = torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _empty(cache, shape):
    if cache == "f16":
        return (torch.zeros(shape, dtype=torch.float16, device="cuda"),)
    return (torch.zeros(*shape[:-1], shape[-1] // 2, dtype=torch.uint8, device="cuda"),
            torch.zeros(*shape[:-1], shape[-1] // CHUNK, dtype=torch.float16, device="cuda"))


def _store(case, cache, table, seq, pos, x):
    """Rows x, in 64 bits, to the slots of their positions."""
    page, slot = table.long()[seq, pos // case["page"]], pos % case["page"]
    x = x.float()
    if case["cache"] == "f16":
        cache[0][page, slot] = x.half()
        return
    b = x.unflatten(-1, (-1, CHUNK))
    size = b.abs()
    lane = torch.arange(CHUNK, device="cuda")
    first = torch.where(size == size.amax(-1, keepdim=True), lane, CHUNK).amin(-1, keepdim=True)
    d = (b.gather(-1, first) * -0.125).half()
    code = torch.floor(b.double() / d.double() + 8.5).clamp(0, 15)
    code = torch.where(d == 0, 8, code).to(torch.uint8).flatten(-2)
    cache[0][page, slot] = code[..., 0::2] | (code[..., 1::2] << 4)
    cache[1][page, slot] = d[..., 0]


def _values(case, cache, *at):
    """The cached values at [at], in 32 bits."""
    if case["cache"] == "f16":
        return cache[0][at].float()
    code, d = cache[0][at], cache[1][at].float()
    code = torch.stack([code & 15, code >> 4], -1).flatten(-2).float() - 8
    return (code.unflatten(-1, (-1, CHUNK)) * d[..., None]).flatten(-2)


def _plain_rotate(state):
    case = state["case"]
    cs = state["table"][state["positions"].long()]
    out = []
    for x, w in ((state["q"], state.get("q_norm")), (state["k"], state.get("k_norm"))):
        x = x.float()
        out.append(_rotate(_rms(x, w) if w is not None else x, cs, case["half"]).to(TYPES[case["output"]]))
    return out


def _plain_read(state, dtype):
    case = state["case"]
    seq, pos = state["where"]
    page, slot = state["page_table"].long()[seq, pos // case["page"]], pos % case["page"]
    return [_values(case, c, page, slot).to(dtype) for c in state["cache"]]


def _plain_append(state):
    case = state["case"]
    seq, pos = state["where"]
    k = state["k"].double()  # in 64 bits: a code next to a border does not hang on the order of the sums
    if "k_norm" in state:
        k = _rms(k, state["k_norm"])
    k = _rotate(k, state["table"][pos], case["half"])
    _store(case, state["cache"][0], state["page_table"], seq, pos, k)
    _store(case, state["cache"][1], state["page_table"], seq, pos, state["v"].double())
    return _plain_read(state, torch.float16)


def _plain_attend(state):
    case, q = state["case"], state["q"]
    n, heads, dim = q.shape
    kvh = case["kv_heads"]
    group = heads // kvh
    seq, pos = state["where"]
    seqs, most = case["seqs"], case["rows"]
    table = state["page_table"].long()
    k, v = (_values(case, c, table).flatten(1, 2).transpose(1, 2) for c in state["cache"])  # [seqs, kvh, positions, dim]
    j = torch.arange(n, device="cuda") - state["row_start"].long()[seq]
    qs = torch.zeros(seqs, kvh, most, group, dim, device="cuda")
    qs[seq, :, j] = q.float().unflatten(1, (kvh, group))
    at = torch.full((seqs, most), -1, device="cuda")
    at[seq, j] = pos
    x = torch.arange(k.shape[2], device="cuda")
    seen = x <= at[:, :, None]
    if case["window"]:
        seen &= x > at[:, :, None] - case["window"]
    s = (qs.flatten(2, 3) * (1 / math.sqrt(dim))) @ k.transpose(2, 3).contiguous()
    s = s.unflatten(2, (most, group)).masked_fill_(~seen[:, None, :, None], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    o = (s.flatten(2, 3) @ v.contiguous()).unflatten(2, (most, group)) / torch.where(total > 0, total, 1)
    return o[seq, :, j].flatten(1, 2).to(q.dtype)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state)
    if kind == "rotate":
        return _plain_rotate(state)
    if kind == "append":
        return _plain_append(state)
    if kind == "read":
        return _plain_read(state, TYPES[state["case"]["output"]])
    return _plain_attend(state)


# ---------------------------------------------------------------- the library's calls

def _heads(L, x):
    """A [rows, heads, dim] tensor as the library takes it."""
    return L.HipHeads(x.data_ptr(), GGML[{v: k for k, v in TYPES.items()}[x.dtype]], x.stride(0), x.stride(1))


def _prepare_own(state):
    """The cache and the argument blocks that a program keeps."""
    if "brisk-llm_amd" not in sys.path:
        sys.path.insert(0, "brisk-llm_amd")
    from brisk_hip import lib as L
    case, lib = state["case"], L.load()
    state["lib"], state["check"] = lib, L.check
    dim, kvh = case["head_dim"], case["kv_heads"]
    ref = {}
    if "table" in state:
        ref["rope"] = L.HipRope(state["table"].data_ptr(), state["table"].shape[0], case["rotated"], 1 if case["half"] else 2)
    if case["kind"] == "rotate":
        kind = TYPES[case["output"]]
        state["out"] = [torch.empty(x.shape, dtype=kind, device="cuda") for x in (state["q"], state["k"])]
        ref["q"], ref["k"] = _heads(L, state["q"]), _heads(L, state["k"])
        ref["q_out"], ref["k_out"] = (_heads(L, x) for x in state["out"])
    else:
        rows, lengths = _batch(case)
        kv = L.HipKv(None, GGML[case["cache"]], kvh, dim, case["page"], state["pages"])
        state["memory"] = torch.empty(lib.brisk_hip_kv_bytes(C.byref(kv)), dtype=torch.uint8, device="cuda")
        kv.data = state["memory"].data_ptr()
        ref["kv"] = kv

        def batch(starts, n, most):
            return L.HipBatch(starts.data_ptr(), state["lengths"].data_ptr(), state["page_table"].data_ptr(), len(rows), n,
                              state["page_table"].stride(0), most, max(lengths))

        ref["batch"] = batch(state["row_start"], sum(rows), max(rows))
        if case["kind"] != "append":  # what earlier steps have stored
            k, v, all_ = _heads(L, state["k"]), _heads(L, state["v"]), batch(state["stored"], state["k"].shape[0], max(lengths))
            L.check(lib.brisk_hip_kv_append(C.byref(kv), C.byref(all_), C.byref(k), C.byref(v), None, 0.0, None, _stream()))
            torch.cuda.synchronize()
            del state["k"], state["v"]
        else:
            ref["k"], ref["v"] = _heads(L, state["k"]), _heads(L, state["v"])
        if case["kind"] == "attend":
            state["out"] = torch.empty_like(state["q"])
            ref["q"], ref["out"] = _heads(L, state["q"]), _heads(L, state["out"])
            size = lib.brisk_hip_paged_attention_bytes(C.byref(kv), C.byref(ref["batch"]), case["heads"])
            state["workspace"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
        else:
            kind = TYPES[case.get("output", "f16")]
            state["out"] = [torch.empty(sum(rows), kvh, dim, dtype=kind, device="cuda") for _ in range(2)]
            ref["k_out"], ref["v_out"] = (_heads(L, x) for x in state["out"])
    state["refs"] = ref  # (kept alive)
    state["by"] = {name: C.byref(x) for name, x in ref.items()}


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _pointer(state, name):
    return state[name].data_ptr() if name in state else None


def _run_own(state):
    case, lib, check, by = state["case"], state["lib"], state["check"], state["by"]
    kind = case["kind"]
    if kind == "rotate":
        check(lib.brisk_hip_qk_norm_rope(by["q"], by["k"], case["n"], case["heads"], case["kv_heads"], case["head_dim"], _pointer(state, "q_norm"),
                                         _pointer(state, "k_norm"), EPS, by["rope"], state["positions"].data_ptr(), by["q_out"], by["k_out"], _stream()))
    elif kind == "attend":
        check(lib.brisk_hip_paged_attention(by["kv"], by["batch"], by["q"], case["heads"], 1 / math.sqrt(case["head_dim"]), case["window"], by["out"],
                                            state["workspace"].data_ptr(), state["workspace"].numel(), _stream()))
    else:
        if kind == "append":
            check(lib.brisk_hip_kv_append(by["kv"], by["batch"], by["k"], by["v"], _pointer(state, "k_norm"), EPS, by["rope"], _stream()))
        check(lib.brisk_hip_kv_read(by["kv"], by["batch"], by["k_out"], by["v_out"], _stream()))
    return state["out"]


# ---------------------------------------------------------------- what a pass costs, and what it should give

def _row_bytes(cache, dim):
    return 2 * dim if cache == "f16" else dim // 2 + dim // 16


def work(case):
    dim, kvh = case["head_dim"], case["kv_heads"]
    if case["kind"] == "rotate":
        values = case["n"] * (case["heads"] + kvh) * dim
        return {"bytes": values * (SIZES[case["input"]] + SIZES[case["output"]]) + case["n"] * (4 * case["rotated"] + 4),
                "flops": values * (6 if case["norm"] else 3)}
    rows, lengths = _batch(case)
    n, cached = sum(rows), _row_bytes(case["cache"], dim)
    if case["kind"] == "append":
        values = 2 * n * kvh * dim
        return {"bytes": values * (SIZES[case["input"]] + 2) + 2 * n * kvh * cached + n * 4 * case["rotated"], "flops": 8 * values}
    if case["kind"] == "read":
        return {"bytes": 2 * n * kvh * (cached + dim * SIZES[case["output"]]), "flops": 2 * n * kvh * dim}
    window = case["window"] or 1 << 60
    read = sum(min(l, r - 1 + window) for r, l in zip(rows, lengths))
    pairs = sum(min(window, l - r + 1 + j) for r, l in zip(rows, lengths) for j in range(r))
    return {"bytes": 2 * n * case["heads"] * dim * SIZES[case["input"]] + 2 * read * kvh * cached, "flops": 4 * pairs * case["heads"] * dim}


def _exact_turn(x, w, table, positions, rotated, half):
    """The definition pair by pair: complex numbers times the position's unit."""
    x = x.double().clone()
    if w is not None:
        x = w.double() * x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    i = torch.arange(rotated // 2, device="cuda")
    first, second = (i, i + rotated // 2) if half else (2 * i, 2 * i + 1)
    unit = torch.view_as_complex(table.double()[positions.long()].contiguous())[:, None]
    z = torch.complex(x[..., first], x[..., second]) * unit
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_held(cache, x):
    """What a cache that holds rows x (64 bits, read as 32) stands for."""
    x = x.float()
    if cache == "f16":
        return x.half().double()
    b = x.reshape(-1, CHUNK).cpu().numpy()
    top = b[np.arange(len(b)), np.abs(b).argmax(1)]  # numpy's argmax is the first of equals
    d = (top / np.float32(-8)).astype(np.float16).astype(np.float64)[:, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.minimum(np.floor(b.astype(np.float64) / d + 8.5), 15) - 8
    return torch.from_numpy(np.where(d == 0, 0, code * d)).reshape(x.shape).cuda()


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "rotate":
        return [_exact_turn(d[x], d.get(x + "_norm"), d["table"], d["positions"], case["rotated"], case["half"]) for x in ("q", "k")]
    rows, lengths = _batch(case)
    if case["kind"] == "read":
        return [_exact_held(case["cache"], d[x]) for x in ("k", "v")]
    if case["kind"] == "append":
        positions = torch.cat([torch.arange(l - r, l) for r, l in zip(rows, lengths)]).cuda()
        k = _exact_turn(d["k"], d.get("k_norm"), d["table"], positions, case["rotated"], case["half"])
        return [_exact_held(case["cache"], k), _exact_held(case["cache"], d["v"].double())]
    k, v = _exact_held(case["cache"], d["k"]), _exact_held(case["cache"], d["v"])
    q, out = d["q"].double(), []
    group, t, at = case["heads"] // case["kv_heads"], 0, 0
    for r, l in zip(rows, lengths):
        here = torch.arange(l - r, l, device="cuda")[:, None]
        there = torch.arange(l, device="cuda")[None]
        hidden = there > here
        if case["window"]:
            hidden |= there <= here - case["window"]
        heads = []
        for h in range(case["heads"]):
            s = q[at:at + r, h] @ k[t:t + l, h // group].T.contiguous() / math.sqrt(case["head_dim"])
            heads.append(torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[t:t + l, h // group])
        out.append(torch.stack(heads, 1))
        t, at = t + l, at + r
    return torch.cat(out)
