"""The paged-cache operators on the GPU against their plain forms in 64 bits (tests/paged_reference.py).

Tolerances count roundings.  A result of type t is off by half a step of t.  Norms and rotations in 32 bits: a value passes
fewer than 16 roundings of 2^-24, of terms no larger than the pair's.  Attention in 16 bits: a probability is rounded to 16 bits (2^-11 of
it) and so is a 4-bit value's product with its scale (2^-11), so a result is off by at most 2^-10 sum p |v|; a score, whose terms are
exact products summed in 32 bits with at most dim / 8 roundings on a path, by e = dim / 8 2^-24 sum |q| |k| scale, which changes a
probability by at most 2 e of it, as the exponential's own error (2^-21) does; the sums over L positions add L / 16 + 32 roundings of
2^-24.  In 32 bits the queries and probabilities are sums of two 16-bit parts: 2^-21 in the place of 2^-10, and twice
the score's terms, with 2^-21 of sum |q| |k| scale for the query's own remainder.  A probability next to 0 is held in a half's smallest
steps, 2^-24 where the largest is at least 2^7: off by half a step, 2^-32 of the largest, which is at most 1, so 2^-32 sum |v| in all.  Prompts' 4-bit
keys are rounded to 16 bits as their values are, each by at most 2^-11 of it and independently: by Hoeffding's bound a score is off by
more than 7.5 2^-11 sqrt(sum (q k scale)^2) once in 10^12.
"""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from brisk_hip import lib as L  # noqa: E402
import paged_reference as R  # noqa: E402
from paged_reference import BF16, F16, F32, HALF_STEP, Q4_0, Batch  # noqa: E402

TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
NAMES = {F32: "f32", F16: "f16", BF16: "bf16", Q4_0: "q4_0"}


@pytest.fixture(scope="module")
def lib():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return L.load()


@pytest.fixture(params=["lengths", "wide"])
def tables(request):
    """The host knows the lengths, or only that the tables have room for 2^20 positions: then there are more parts, and
    prompts go to the kernel of many columns."""
    Cache.wide_tables = request.param == "wide"
    yield
    Cache.wide_tables = False


def heads_of(x):
    return L.HipHeads(x.data_ptr(), {v: k for k, v in TORCH.items()}[x.dtype], x.stride(0), x.stride(1))


def ref(x):
    return C.byref(x) if x is not None else None


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def ptr(t):
    return None if t is None else t.data_ptr()


def rows(rng, n, heads, dim, kind, scale=1.0):
    return torch.from_numpy((rng.standard_normal((n, heads, dim)) * scale).astype(np.float32)).to(TORCH[kind])


def host(t):
    torch.cuda.synchronize()
    return t.detach().cpu().double().numpy()


class Cache:
    """A cache and a batch on the GPU.  The cache's bytes start as 0xFF, which read as NaN."""
    wide_tables = False

    def __init__(self, lib, batch, kind, kv_heads, dim, max_rows=None, max_length=None, extra_rows=0):
        self.lib, self.batch, self.kind = lib, batch, kind
        self.kv = L.HipKv(None, kind, kv_heads, dim, batch.page, batch.pages)
        size = lib.brisk_hip_kv_bytes(C.byref(self.kv))
        assert size > 0
        self.memory = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        self.kv.data = self.memory.data_ptr()
        self.max_rows = max(batch.rows + [0]) if max_rows is None else max_rows
        self.max_length = max(max(batch.lengths), 0) if max_length is None else max_length
        self.extra = extra_rows
        self.set(batch)

    def set(self, batch):
        self.batch = batch
        table, length = batch.table, self.max_length
        if Cache.wide_tables:
            table, length = np.pad(table, ((0, 0), (0, (1 << 20) // batch.page - table.shape[1])), constant_values=-1), 0
        self.arrays = [torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda() for a in (batch.starts, batch.lengths, table)]
        stride = table.shape[1] if Cache.wide_tables else batch.stride
        self.b = L.HipBatch(*[a.data_ptr() for a in self.arrays], len(batch.rows), batch.n + self.extra, stride, self.max_rows, length)

    def append(self, k, v, w=None, eps=1e-6, rope=None):
        kh, vh = heads_of(k), heads_of(v)
        L.check(self.lib.brisk_hip_kv_append(ref(self.kv), ref(self.b), ref(kh), ref(vh), ptr(w), eps, ref(rope), stream()))

    def read(self, kind=F32, fill=0.0):
        out = [torch.full((self.b.rows, self.kv.kv_heads, self.kv.head_dim), fill, dtype=TORCH[kind], device="cuda") for _ in range(2)]
        k, v = map(heads_of, out)
        L.check(self.lib.brisk_hip_kv_read(ref(self.kv), ref(self.b), ref(k), ref(v), stream()))
        return out

    def workspace(self, heads):
        return torch.empty(max(16, self.lib.brisk_hip_paged_attention_bytes(ref(self.kv), ref(self.b), heads)), dtype=torch.uint8, device="cuda")

    def attend(self, q, scale, window=0, out=None, work=None):
        out = torch.full_like(q, 7.0) if out is None else out
        work = self.workspace(q.shape[1]) if work is None else work
        qh, oh = heads_of(q), heads_of(out)
        L.check(self.lib.brisk_hip_paged_attention(ref(self.kv), ref(self.b), ref(qh), q.shape[1], scale, window, ref(oh), work.data_ptr(),
                                                   work.numel(), stream()))
        return out


# ---------------------------------------------------------------- norms and rotations

@pytest.mark.parametrize("dim,dims,neox", [(64, 64, 1), (64, 64, 2), (96, 96, 1), (96, 72, 2), (128, 32, 1), (128, 20, 1), (256, 64, 1), (512, 512, 2), (8, 2, 2), (40, 12, 1)])
@pytest.mark.parametrize("kind,out,norm", [(F32, F16, True), (F16, F32, True), (BF16, BF16, False), (F32, F32, False)])
def test_norm_rope(lib, dim, dims, neox, kind, out, norm):
    rng = np.random.default_rng(dim + dims)
    n, heads, kvh, context = 37, 6, 2, 700
    fused = rows(rng, n, heads + 2 * kvh, dim, kind, 2.0).cuda()  # rows as a fused projection leaves them
    q, k = fused[:, :heads], fused[:, heads:heads + kvh]
    w = [torch.from_numpy((1 + 0.3 * rng.standard_normal(dim)).astype(np.float32)).cuda() if norm else None for _ in range(2)]
    table = R.rope_table(context, dims)
    positions = rng.integers(0, context, n).astype(np.int32)
    positions[0], positions[1], positions[5], positions[9] = 0, context - 1, -1, context  # the last two: padding
    td, pd = torch.from_numpy(table).cuda(), torch.from_numpy(positions).cuda()
    rope = L.HipRope(td.data_ptr(), context, dims, neox)
    outs = [torch.full((n, h, dim), 5.0, dtype=TORCH[out], device="cuda") for h in (heads, kvh)]
    args = [heads_of(x) for x in (q, k, *outs)]
    L.check(lib.brisk_hip_qk_norm_rope(ref(args[0]), ref(args[1]), n, heads, kvh, dim, ptr(w[0]), ptr(w[1]), 1e-6, ref(rope), pd.data_ptr(),
                                       ref(args[2]), ref(args[3]), stream()))
    live = (positions >= 0) & (positions < context)
    for x, wt, y in zip((q, k), w, outs):
        want = R.norm_rope(host(x), None if wt is None else host(wt), 1e-6, table, np.where(live, positions, 0), dims, neox)
        got = host(y)
        assert (got[~live] == 5.0).all()
        size = np.abs(want).max(-1, keepdims=True) * 1.5  # a pair's terms are at most sqrt(2) of its largest value
        assert (np.abs(got - want)[live] <= (HALF_STEP[out] * np.abs(want) + 16 * 2.0 ** -24 * size)[live]).all()


def test_norm_rope_in_place_unaligned_and_queries_alone(lib):
    rng = np.random.default_rng(3)
    n, heads, dim = 5, 3, 64
    base = torch.zeros(n * heads * dim + 1, dtype=torch.float16, device="cuda")
    x = base[1:].view(n, heads, dim)  # two bytes past a 16-byte border
    x.copy_(rows(rng, n, heads, dim, F16))
    before = host(x)
    table, positions = R.rope_table(50, dim), np.arange(n, dtype=np.int32) * 7
    td, pd = torch.from_numpy(table).cuda(), torch.from_numpy(positions).cuda()
    rope, a = L.HipRope(td.data_ptr(), 50, dim, 1), heads_of(x)
    L.check(lib.brisk_hip_qk_norm_rope(ref(a), None, n, heads, 0, dim, None, None, 0.0, ref(rope), pd.data_ptr(), ref(a), None, stream()))
    want = R.norm_rope(before, None, 0, table, positions, dim, 1)
    assert (np.abs(host(x) - want) <= HALF_STEP[F16] * np.abs(want) + 16 * 2.0 ** -24 * np.abs(want).max()).all()
    # no rotation: norms alone, without positions
    w = torch.ones(dim, device="cuda")
    y = torch.empty(n, heads, dim, device="cuda")
    b = heads_of(y)
    L.check(lib.brisk_hip_qk_norm_rope(ref(a), None, n, heads, 0, dim, w.data_ptr(), None, 1e-6, None, None, ref(b), None, stream()))
    want = R.norm_rope(host(x), np.ones(dim), 1e-6, None, None, 0, 1)
    assert (np.abs(host(y) - want) <= 16 * 2.0 ** -24 * np.abs(want).max()).all()


# ---------------------------------------------------------------- the cache's rows

def check_held(got, x, kind, normed):
    """Cached rows are exactly what their type stands for; where norms (not exact in 64 bits) put a value within 2^-20 of a border
    the neighbouring code is right too."""
    want, near = R.held(x, kind)
    if normed and kind == F16:
        assert (np.abs(got - want) <= 2.0 ** -10 * np.abs(want)).all() and (got != want).mean() < 1e-3
        return
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    if normed:
        bad &= near > 2.0 ** -20
    assert not bad.any()


@pytest.mark.parametrize("kind", [F16, Q4_0], ids=NAMES.get)
@pytest.mark.parametrize("dim,dims,neox,norm,src", [(64, 64, 2, False, F32), (96, 48, 1, True, BF16), (128, 128, 1, True, F32), (256, 64, 1, False, F16),
                                                    (512, 512, 2, True, F32), (128, 24, 1, False, F32)])
@pytest.mark.parametrize("page", [16, 64])
def test_append_and_read(lib, kind, dim, dims, neox, norm, src, page):
    rng = np.random.default_rng(dim + page)
    kvh = 3
    batch = Batch([1, 40, 0, 17, 5], [33, 77, 9, 17, 64], page, seed=dim)
    cache = Cache(lib, batch, kind, kvh, dim)
    fused = rows(rng, batch.n, 2 * kvh + 1, dim, src).cuda()
    k, v = fused[:, 1:1 + kvh], fused[:, 1 + kvh:]
    w = torch.from_numpy((1 + 0.3 * rng.standard_normal(dim)).astype(np.float32)).cuda() if norm else None
    table = R.rope_table(100, dims)
    td = torch.from_numpy(table).cuda()
    cache.append(k, v, w, 1e-6, L.HipRope(td.data_ptr(), 100, dims, neox))
    kk, vv = cache.read()
    want = R.norm_rope(host(k), None if w is None else host(w), 1e-6, table, batch.positions(), dims, neox)
    check_held(host(kk), want, kind, norm)
    check_held(host(vv), host(v), kind, False)
    for out in (F16, BF16):  # the same rows in other types
        for a, b in zip(cache.read(out), (kk, vv)):
            assert (host(a) == host(b.to(TORCH[out]))).all()
    # nothing else was written: a fresh cache with the same rows has the same bytes, and the rest is as it was
    touched = (cache.memory != 255).sum().item()
    assert touched <= 2 * batch.n * kvh * (2 * dim if kind == F16 else dim // 2 + dim // 16)
    # rows of positions before the appended ones are still unset: they read as NaN
    earlier = Batch([32, 37, 9, 0, 59], [32, 37, 9, 0, 59], page, seed=dim)
    earlier.table, earlier.stride = batch.table, batch.stride
    cache.set(earlier)
    assert np.isnan(host(cache.read()[0])).all()


@pytest.mark.parametrize("kind", [F16, Q4_0], ids=NAMES.get)
@pytest.mark.parametrize("dim,dims,neox,norm,src", [(64, 16, 1, True, F32), (64, 20, 1, False, F16), (64, 2, 1, True, F32), (96, 24, 1, True, F16), (96, 96, 1, False, BF16), (128, 32, 1, True, BF16),
                                                    (128, 100, 1, True, F32), (128, 112, 1, False, F32), (128, 64, 1, True, F16), (256, 128, 1, True, F32), (256, 96, 1, True, F16),
                                                    (512, 256, 1, True, BF16), (512, 20, 1, False, F32), (128, 40, 2, True, F32), (96, 20, 2, False, F16), (256, 2, 2, True, F32)])
def test_append_rotations(lib, kind, dim, dims, neox, norm, src):
    """Pairs in a lane, in others, in other blocks; part of the head; tables whose rows are not 16-byte aligned."""
    test_append_and_read(lib, kind, dim, dims, neox, norm, src, 32)


@pytest.mark.parametrize("kind", [F16, Q4_0], ids=NAMES.get)
def test_append_special_values(lib, kind):
    """Zero blocks, ties, equal magnitudes of either sign, subnormal scales, infinities, NaN, values past 16 bits."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, 1, 64)).astype(np.float32)
    x[0] = 0
    x[1, 0, :32] = np.arange(32) - 15.5
    x[2, 0, 3], x[2, 0, 9], x[2, 0, 20] = -4, 4, -4
    x[3, 0, 3], x[3, 0, 9] = 4, -4
    x[4] *= 1e-7
    x[5] *= 3e-6
    x[6, 0, 40] = np.inf
    x[7, 0, 2] = np.nan
    x[8, 0, 2] = -np.inf
    x[9, 0, 50] = 7e4
    x[10, 0, 50] = 6e5
    x[10, 0, 5] = 65500
    x[11, 0, :32] = -0.0
    batch = Batch([12], [12], 16)
    cache = Cache(lib, batch, kind, 1, 64)
    t = torch.from_numpy(x).cuda()
    cache.append(t, t)
    for y in cache.read():
        check_held(host(y), x.astype(np.float64), kind, False)


def test_append_leaves_out_what_has_no_place(lib):
    """Rows before position 0, past the table, on entries that are no page, past the rotation's table, and rows of no sequence."""
    batch = Batch([5, 20, 3, 6], [3, 20, 3, 40], 16, spare=0)
    batch.table[1, 1] = -1                  # positions 16..19 of sequence 1
    batch.table[2, 0] = batch.pages         # one past the pool
    cache = Cache(lib, batch, F16, 2, 64, extra_rows=4)
    rng = np.random.default_rng(1)
    k = rows(rng, batch.n + 4, 2, 64, F32).cuda()
    table = R.rope_table(38, 64)
    td = torch.from_numpy(table).cuda()
    cache.append(k, k, rope=L.HipRope(td.data_ptr(), 38, 64, 1))
    kk, vv = (host(x) for x in cache.read(F32, fill=9.0))
    pos = batch.positions()
    stored = np.zeros(batch.n + 4, bool)
    stored[2:5], stored[5:21], stored[28:32] = True, True, True
    seen = stored.copy()
    seen[32:34] = True  # positions 38 and 39 have a page, but no rotation: never written
    assert (vv[~seen] == 9.0).all() and (kk[~seen] == 9.0).all()
    assert np.isnan(vv[32:34]).all()
    check_held(vv[stored], host(k)[stored], F16, False)
    check_held(kk[stored], R.norm_rope(host(k)[:batch.n][stored[:batch.n]], None, 0, table, pos[stored[:batch.n]], 64, 1), F16, False)


def test_rows_by_head_and_sessions_layout(lib):
    """Rows laid out as a session's cache, [kv_head][context][head_dim] in fp16, in and out."""
    batch = Batch([50], [50], 32)
    src = torch.randn(2, 80, 128, dtype=torch.float16, device="cuda")
    dst = torch.zeros_like(src)
    cache = Cache(lib, batch, F16, 2, 128)
    a = L.HipHeads(src.data_ptr(), F16, 128, 80 * 128)
    b = L.HipHeads(dst.data_ptr(), F16, 128, 80 * 128)
    L.check(lib.brisk_hip_kv_append(ref(cache.kv), ref(cache.b), ref(a), ref(a), None, 0.0, None, stream()))
    L.check(lib.brisk_hip_kv_read(ref(cache.kv), ref(cache.b), None, ref(b), stream()))
    assert torch.equal(dst[:, :50], src[:, :50]) and (dst[:, 50:] == 0).all()


def test_cache_past_32_bits(lib):
    """A pool of over 4 GiB, the sequences on its last and its first page."""
    batch = Batch([40], [40], 64, pool=33000)
    batch.table[0, 0] = batch.pages - 1
    cache = Cache(lib, batch, F16, 8, 64)
    assert cache.memory.numel() > 1 << 32
    k = torch.randn(40, 8, 64, device="cuda").half()
    cache.append(k, 2 * k)
    kk, vv = cache.read(F16)
    assert torch.equal(kk, k) and torch.equal(vv, 2 * k)
    q = torch.randn(40, 8, 64, device="cuda").half()
    check_attention(cache, q, cache.attend(q, 0.125), 0.125, 0)


# ---------------------------------------------------------------- attention

def whole(cache):
    """Every position of every sequence, as the cache holds it (64 bits), and which there are."""
    b = cache.batch
    every = Batch(b.lengths, b.lengths, b.page)
    every.table, every.stride, every.pages = b.table, b.stride, b.pages
    extra, cache.extra = cache.extra, 0
    cache.set(every)
    k, v = (host(x) for x in cache.read(F32, fill=np.nan))
    cache.extra = extra
    cache.set(b)
    there = [np.repeat((b.table[s] >= 0) & (b.table[s] < b.pages), b.page)[:l] for s, l in enumerate(b.lengths)]
    return k, v, every.starts, there


def check_attention(cache, q, out, scale, window, kv=None):
    b = cache.batch
    k, v, starts, there = kv or whole(cache)
    qq, got = host(q), host(out)
    kind = {v: k for k, v in TORCH.items()}[out.dtype]
    exact = q.dtype == torch.float32 or out.dtype == torch.float32
    for s, (r, l) in enumerate(zip(b.rows, b.lengths)):
        mine = slice(b.starts[s], b.starts[s] + r)
        at = slice(starts[s], starts[s] + max(l, 0))
        want, mass, size, total, spread = R.attend(qq[mine], k[at], v[at], np.arange(l - r, l), there[s], float(np.float32(scale)), window)
        dim = q.shape[2]
        score = (dim / 8 * (2 if exact else 1) * 2.0 ** -24 + (2.0 ** -21 if exact else 0)) * size
        if cache.kind == Q4_0 and not exact and r > 8:
            score = score + 7.5 * 2.0 ** -11 * spread
        tol = HALF_STEP[kind] * np.abs(want) + mass * ((2.0 ** -21 if exact else 2.0 ** -10) + 2 * score + 2.0 ** -20 + (l / 16 + 32) * 2.0 ** -24) + 2.0 ** -32 * total
        fine = np.isfinite(want)
        assert (np.isnan(got[mine]) == np.isnan(want)).all(), f"sequence {s}: NaN"
        assert (got[mine][~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all()
        off = np.abs(got[mine] - want)
        assert (off[fine] <= tol[fine] + 1e-30).all(), f"sequence {s}: {np.nanmax(np.where(fine, off / (tol + 1e-30), 0))} of the tolerance"


def filled(lib, batch, kind, kvh, dim, seed=0, **more):
    """A cache with every position of the batch's sequences appended (float16 rows, some dimensions large)."""
    rng = np.random.default_rng(seed)
    cache = Cache(lib, batch, kind, kvh, dim, **more)
    every = Batch([max(l, 0) for l in batch.lengths], batch.lengths, batch.page)
    every.table, every.stride, every.pages = batch.table, batch.stride, batch.pages
    cache.max_rows, extra, cache.extra = 0, cache.extra, 0
    cache.set(every)
    if every.n:
        k = rows(rng, every.n, kvh, dim, F16)
        k *= torch.from_numpy(np.exp(0.5 * rng.standard_normal((kvh, dim)))).half()
        cache.append(k.cuda(), rows(rng, every.n, kvh, dim, F16).cuda())
    cache.extra = extra
    cache.max_rows = max(batch.rows + [0]) if more.get("max_rows") is None else more["max_rows"]
    cache.set(batch)
    return cache


LENGTHS = [([1, 1, 1, 1], [1, 17, 700, 1300]), ([3, 8, 1], [40, 8, 333]), ([70, 33], [200, 33]), ([300, 1, 0, 129], [300, 500, 70, 700])]


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("rows_,lengths", LENGTHS, ids=["tokens", "drafted", "prompts", "mixed"])
@pytest.mark.parametrize("kind", [F16, Q4_0], ids=NAMES.get)
@pytest.mark.parametrize("heads,kvh,dim,src", [(16, 8, 128, F16), (4, 1, 64, BF16), (6, 2, 96, F32), (4, 1, 256, F32), (8, 2, 256, F16), (8, 1, 512, F32),
                                               (8, 1, 512, BF16), (20, 5, 128, F32), (32, 1, 64, F16), (3, 3, 128, BF16)])
@pytest.mark.parametrize("page,window", [(16, 0), (128, 100)])
def test_attention(lib, rows_, lengths, kind, heads, kvh, dim, src, page, window):
    batch = Batch(rows_, lengths, page, seed=heads)
    cache = filled(lib, batch, kind, kvh, dim, seed=dim)
    q = rows(np.random.default_rng(7), batch.n, heads, dim, src, 1.3).cuda()
    scale = dim ** -0.5
    check_attention(cache, q, cache.attend(q, scale, window), scale, window)


@pytest.mark.parametrize("kind", [F16, Q4_0], ids=NAMES.get)
@pytest.mark.parametrize("src", [F16, F32], ids=NAMES.get)
def test_attention_long(lib, kind, src):
    """Positions split between many workgroups, a length that ends inside a tile, and a short one beside it."""
    batch = Batch([1, 2], [20011, 35], 64)
    cache = filled(lib, batch, kind, 2, 128)
    q = rows(np.random.default_rng(9), 3, 8, 128, src, 2.0).cuda()
    check_attention(cache, q, cache.attend(q, 0.0884), 0.0884, 0)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("kind", [F16, Q4_0], ids=NAMES.get)
@pytest.mark.parametrize("rows_", [[1, 4, 9, 0, 2], [30, 64, 50, 0, 40]], ids=["few", "many"])
def test_attention_rows_that_see_nothing(lib, kind, rows_):
    """No length, more rows than positions, no rows, entries that are no page, rows of no sequence."""
    batch = Batch(rows_, [0, 2, 30, 5, 40], 16)
    batch.table[2, 0] = -1
    batch.table[4, 1], batch.table[4, 2] = batch.pages, -5
    cache = filled(lib, batch, kind, 2, 64, extra_rows=3)
    q = rows(np.random.default_rng(2), batch.n + 3, 4, 64, F16).cuda()
    out = cache.attend(q, 0.125)
    check_attention(cache, q, out, 0.125, 0)
    got = host(out)
    assert (got[:rows_[0]] == 0).all() and (got[batch.n:] == 7.0).all()
    cache = filled(lib, batch, kind, 2, 64, extra_rows=3)
    out = cache.attend(q, 0.125, 3)  # a window all of whose positions are missing
    check_attention(cache, q, out, 0.125, 3)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("kind", [F16, Q4_0], ids=NAMES.get)
@pytest.mark.parametrize("src", [F16, F32], ids=NAMES.get)
@pytest.mark.parametrize("rows_", [3, 40])
@pytest.mark.parametrize("byte", [0xFF, 0x7C, 0x7B, 0x72, 0xFB])
def test_attention_over_memory_never_written(lib, kind, src, rows_, byte):
    """What lies behind a sequence's end in its last page, whatever it is, has no part in the result."""
    batch = Batch([rows_], [77], 64)
    cache = Cache(lib, batch, kind, 1, 64)
    cache.memory.fill_(byte)
    x = torch.randn(77, 1, 64, device="cuda")
    every = Batch([77], [77], 64)
    every.table, every.pages = batch.table, batch.pages
    cache.max_rows = 0
    cache.set(every)
    cache.append(x, x.flip(0))
    cache.set(batch)
    q = rows(np.random.default_rng(2), rows_, 3, 64, src).cuda()
    check_attention(cache, q, cache.attend(q, 0.125), 0.125, 0)


@pytest.mark.parametrize("hints", [(0, 0), (1, 1), (500, 100000), (2, 5)])
def test_attention_does_not_depend_on_the_hosts_bounds(lib, hints):
    batch = Batch([3, 40, 1], [30, 90, 400], 32)
    cache = filled(lib, batch, Q4_0, 2, 64, max_rows=hints[0], max_length=hints[1])
    q = rows(np.random.default_rng(2), batch.n, 8, 64, F16).cuda()
    check_attention(cache, q, cache.attend(q, 0.125), 0.125, 0)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("kind", [F16, Q4_0], ids=NAMES.get)
@pytest.mark.parametrize("src", [F16, F32], ids=NAMES.get)
@pytest.mark.parametrize("rows_", [6, 60])
@pytest.mark.parametrize("window", [0, 20])
def test_attention_values_that_are_not_finite(lib, kind, src, rows_, window):
    """Infinities and NaN in values and keys: rows that do not see their position are as if they were not there."""
    batch = Batch([rows_], [100], 16)
    cache = Cache(lib, batch, kind, 1, 64, max_rows=0)
    rng = np.random.default_rng(4)
    k, v = rng.standard_normal((2, 100, 1, 64)).astype(np.float32)
    v[97, 0, 5], v[95, 0, 40], v[96, 0, 41] = np.inf, np.nan, -np.inf
    v[45, 0, 9], v[99, 0, 63] = -np.inf, np.inf
    k[98, 0, 3] = np.nan
    every = Batch([100], [100], 16)
    every.table, every.pages = batch.table, batch.pages
    cache.set(every)
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    cache.set(batch)
    q = rows(rng, rows_, 4, 64, src).cuda()
    out = cache.attend(q, 0.125, window)
    check_attention(cache, q, out, 0.125, window)
    got = host(out)
    if window:  # without one, position 45 is seen
        assert np.isfinite(got[-6]).all()
    assert not np.isfinite(got[-1]).any()  # a NaN key: its row's every value


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("src", [F16, F32], ids=NAMES.get)
@pytest.mark.parametrize("rows_", [1, 200])
def test_attention_infinity_with_a_small_probability(lib, src, rows_):
    """A probability that rounds to 0 times an infinite value: the infinity, as in the formula."""
    batch = Batch([rows_], [300], 16)
    cache = Cache(lib, batch, F16, 1, 64, max_rows=0)
    k, v = np.zeros((300, 1, 64), np.float32), np.ones((300, 1, 64), np.float32)
    k[0], k[1:] = 1, -1
    v[5, 0, 2], v[6, 0, 3] = np.inf, -np.inf
    every = Batch([300], [300], 16)
    every.table, every.pages = batch.table, batch.pages
    cache.set(every)
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    cache.set(batch)
    q = torch.ones(rows_, 2, 64, dtype=TORCH[src], device="cuda")
    got = host(cache.attend(q, 0.35))  # scores of 22.4 and -22.4
    assert (got[:, :, 2] == np.inf).all() and (got[:, :, 3] == -np.inf).all()
    rest = np.delete(got, [2, 3], axis=2)
    assert (np.abs(rest - 1) <= 2.0 ** -9).all()


def test_attention_queries_that_are_not_finite_or_extreme(lib):
    for kind in (F16, Q4_0):
        batch = Batch([1, 1, 1, 1, 1], [50] * 5, 16)
        cache = filled(lib, batch, kind, 1, 64)
        for src in (F32, BF16):
            q = rows(np.random.default_rng(2), 5, 2, 64, src)
            q[0, 0, 3], q[1, 1, 7] = float("inf"), float("nan")
            q[2] *= 1e30
            q[3] *= 1e-38
            q[4] = 0
            q = q.cuda()
            out = cache.attend(q, 1.0)
            got = host(out)
            assert np.isnan(got[0, 0]).all() and np.isnan(got[1, 1]).all() and np.isfinite(got[0, 1]).all() and np.isfinite(got[1, 0]).all()
            k, v, starts, there = whole(cache)
            for r in (3, 4):  # scores next to 0: the mean
                want = v[starts[r]:starts[r] + 50, 0].mean(0)
                assert (np.abs(got[r] - want) <= (2.0 ** -20 + (HALF_STEP[BF16] + 2.0 ** -10 if src == BF16 else 0)) * np.abs(v).max()).all()
            s = k[starts[2]:starts[2] + 50, 0] @ host(q)[2].T
            want = v[starts[2]:starts[2] + 50, 0][s.argmax(0)]  # one score far above the others
            assert (np.abs(got[2] - want) <= (2.0 ** -20 + (HALF_STEP[BF16] + 2.0 ** -10 if src == BF16 else 0)) * np.abs(want) + 1e-30).all()


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("rows_", [2, 200])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30])
def test_attention_scales(lib, rows_, scale):
    """No scale (the mean of what is seen), a negative one, one far below the products."""
    for kind, src in ((F16, F16), (Q4_0, F32)):
        batch = Batch([rows_], [300], 16)
        cache = filled(lib, batch, kind, 2, 64)
        q = rows(np.random.default_rng(2), rows_, 4, 64, src).cuda()
        check_attention(cache, q, cache.attend(q, scale, 50), scale, 50)


@pytest.mark.usefixtures("tables")
def test_attention_strides_types_and_broadcast(lib):
    """Queries inside fused rows, outputs by head, 32-bit outputs of 16-bit queries and the other way round, one query for all heads."""
    batch = Batch([2, 30], [300, 60], 32)
    cache = filled(lib, batch, Q4_0, 2, 128)
    rng = np.random.default_rng(3)
    fused = rows(rng, batch.n, 12, 128, F16).cuda()
    q = fused[:, 2:10]
    for out_kind in (F32, F16, BF16):
        out = torch.zeros(8, batch.n, 128, dtype=TORCH[out_kind], device="cuda").transpose(0, 1)
        cache.attend(q, 0.09, out=out)
        check_attention(cache, q, out, 0.09, 0)
    q = fused.float()[:, :1].expand(batch.n, 8, 128)
    out = torch.zeros(batch.n, 8, 128, dtype=torch.bfloat16, device="cuda")
    cache.attend(q, 0.09, out=out)
    check_attention(cache, q, out, 0.09, 0)
    base = torch.zeros(batch.n * 8 * 128 + 3, dtype=torch.float16, device="cuda")
    q = base[3:].view(batch.n, 8, 128)  # not aligned to 16 bytes
    q.copy_(fused[:, 2:10])
    check_attention(cache, q, cache.attend(q, 0.09), 0.09, 0)


def test_attention_shared_pages_and_repeats(lib):
    """Two sequences on the same prefix pages, one page twice in one sequence, the same call twice with the same bits."""
    batch = Batch([2, 3], [64, 80], 16)
    batch.table[1, :2] = batch.table[0, :2]
    batch.table[1, 3] = batch.table[1, 2]
    cache = filled(lib, batch, F16, 2, 64)
    for r in range(2):  # the appends of shared places race: bring them to one value
        every = Batch([16 * 6], [16 * 6], 16)
    k = torch.randn(16 * batch.pages, 2, 64, device="cuda").half()
    pool = Batch([16 * batch.pages], [16 * batch.pages], 16)
    pool.table, pool.stride, pool.pages = np.arange(batch.pages, dtype=np.int32)[None], batch.pages, batch.pages
    cache.set(pool)
    cache.append(k, k.flip(0))
    cache.set(batch)
    q = rows(np.random.default_rng(2), batch.n, 4, 64, F16).cuda()
    out = cache.attend(q, 0.125)
    check_attention(cache, q, out, 0.125, 0)
    for _ in range(3):
        assert torch.equal(out, cache.attend(q, 0.125))


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("src", [F16, F32], ids=NAMES.get)
@pytest.mark.parametrize("rows_", [[1, 3], [300, 130]], ids=["few", "many"])
def test_attention_into_its_queries(lib, src, rows_):
    """The output in the queries' place: the same bits as beside them."""
    batch = Batch(rows_, [900, 333], 32)
    cache = filled(lib, batch, Q4_0, 2, 128)
    q = rows(np.random.default_rng(5), batch.n, 8, 128, src).cuda()
    want = cache.attend(q, 0.09)
    cache.attend(q, 0.09, out=q)
    assert torch.equal(q, want)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("kind,src,heads,kvh,dim", [(Q4_0, F16, 4, 1, 256), (F16, F32, 4, 2, 64), (Q4_0, BF16, 6, 3, 128)])
def test_attention_of_prompts_captured(lib, kind, src, heads, kvh, dim):
    """A prompt's call captured, and replayed over lengths and tables that changed, with eager calls between: the eager call's bits."""
    batches = [Batch([200, 90], lengths, 16, seed=n, pool=120) for n, lengths in enumerate([[700, 333], [200, 700], [411, 90]])]
    widest = max(b.stride for b in batches)
    for b in batches:
        b.table, b.stride = np.pad(b.table, ((0, 0), (0, widest - b.stride)), constant_values=-1), widest
    cache = Cache(lib, batches[0], kind, kvh, dim, max_rows=200, max_length=700)
    cache.memory.view(torch.float16).copy_(torch.rand(cache.memory.numel() // 2, device="cuda").half())
    q = rows(np.random.default_rng(5), 290, heads, dim, src).cuda()
    out, work = torch.zeros_like(q), cache.workspace(heads)
    cache.attend(q, 0.09, out=out, work=work)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        cache.attend(q, 0.09, out=out, work=work)
    held = cache.arrays
    for b in batches + batches[::-1]:
        cache.set(b)
        want = cache.attend(q, 0.09)
        for mine, new in zip(held, cache.arrays):
            mine.copy_(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---------------------------------------------------------------- together, as a program uses them

@pytest.mark.parametrize("kind", [F16, Q4_0], ids=NAMES.get)
def test_serving_steps_eager_and_captured(lib, kind):
    """Two sequences: a prompt each, then tokens, every step norming, rotating, appending and attending; then the token
    step captured once and replayed on another stream with eager work between, against the same steps in 64 bits."""
    heads, kvh, dim, page, eps, scale = 8, 2, 64, 16, 1e-6, 0.125
    rng = np.random.default_rng(8)
    prompts, steps = [37, 50], 6
    total = [p + steps for p in prompts]
    plan = Batch([0, 0], total, page)
    table = R.rope_table(200, dim)
    td = torch.from_numpy(table).cuda()
    rope = L.HipRope(td.data_ptr(), 200, dim, 1)
    w = [torch.from_numpy((1 + 0.2 * rng.standard_normal(dim)).astype(np.float32)).cuda() for _ in range(2)]
    fused = [[rng.standard_normal((n, heads + 2 * kvh, dim)).astype(np.float32) for n in [p] + [1] * steps] for p in prompts]

    def batch(step):
        lengths = [p + step for p in prompts]
        b = Batch(prompts if step == 0 else [1, 1], lengths, page)
        b.table, b.stride, b.pages = plan.table, plan.stride, plan.pages
        return b

    cache = Cache(lib, batch(0), kind, kvh, dim, max_rows=64, max_length=100)
    n = sum(prompts)
    x = torch.zeros(n, heads + 2 * kvh, dim, device="cuda")
    positions = torch.zeros(n, dtype=torch.int32, device="cuda")
    qr, out = torch.zeros(n, heads, dim, dtype=torch.float16, device="cuda"), torch.zeros(n, heads, dim, device="cuda")

    def step(work):
        b = cache.b
        q, k, v = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]
        a, o = heads_of(q), heads_of(qr)
        L.check(lib.brisk_hip_qk_norm_rope(ref(a), None, b.rows, heads, 0, dim, w[0].data_ptr(), None, eps, ref(rope), positions.data_ptr(), ref(o), None, stream()))
        cache.append(k, v, w[1], eps, rope)
        cache.attend(qr, scale, out=out, work=work)

    def load(i):
        rows_ = np.concatenate([fused[s][i] for s in range(2)])
        x[:len(rows_)].copy_(torch.from_numpy(rows_))
        positions[:len(rows_)].copy_(torch.from_numpy(batch(i).positions().astype(np.int32)))

    def check(i):
        """The step in 64 bits, from the rows so far."""
        b = batch(i)
        got = host(out)
        for s in range(2):
            rows_ = np.concatenate(fused[s][:i + 1])
            pos = np.arange(len(rows_))
            k, _ = R.held(R.norm_rope(rows_[:, heads:heads + kvh], host(w[1]), eps, table, pos, dim, 1), kind)
            v, _ = R.held(rows_[:, heads + kvh:].astype(np.float64), kind)
            q = R.norm_rope(rows_[-b.rows[s]:, :heads], host(w[0]), eps, table, pos[-b.rows[s]:], dim, 1)
            want, mass, size, _, spread = R.attend(q, k, v, pos[-b.rows[s]:], np.ones(len(pos), bool), scale, 0)
            # queries and (16-bit) keys are rounded to 16 bits: 2^-11 of sum |q| |k| scale each, in a score; the cached keys are the same but
            # for those that the norm's last place moves over a border: none of these seeds' values is
            tol = mass * (2 * (2 * 2.0 ** -11) * size + 2.0 ** -19)  # (32-bit outputs: no rounding of 4-bit products)
            assert (np.abs(got[b.starts[s]:b.starts[s + 1]] - want) <= tol).all()

    load(0)
    work = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    step(work)
    check(0)
    for i in (1, 2):
        cache.set(batch(i))
        load(i)
        step(work)
        check(i)
    # captured: the step's arrays are updated in place between the replays
    cache.set(batch(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(work)
    for i in range(3, steps + 1):
        load(i)
        cache.arrays[1].copy_(torch.from_numpy(np.array(batch(i).lengths, np.int32)))
        torch.cuda.synchronize()
        graph.replay()
        check(i)
        replayed = out.clone()
        step(work)  # the same step again, eagerly: the same bits
        torch.cuda.synchronize()
        assert torch.equal(out[:2], replayed[:2])


def test_calls_on_two_streams_at_once(lib):
    """Two caches, two streams, workspaces of their own."""
    sides, checks = [torch.cuda.Stream() for _ in range(2)], []
    caches = [filled(lib, Batch([1], [5000 + s], 32, seed=s), Q4_0, 2, 128, seed=s) for s in range(2)]
    qs = [rows(np.random.default_rng(s), 1, 8, 128, F16).cuda() for s in range(2)]
    works = [c.workspace(8) for c in caches]
    outs = [torch.zeros_like(q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for side, c, q, w, o in zip(sides, caches, qs, works, outs):
            with torch.cuda.stream(side):
                c.attend(q, 0.0884, out=o, work=w)
    torch.cuda.synchronize()
    for c, q, o in zip(caches, qs, outs):
        check_attention(c, q, o, 0.0884, 0)
