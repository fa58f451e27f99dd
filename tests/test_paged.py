"""The paged cache's host side, without a GPU: refusals, sizes, and where a position lies."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from brisk_hip import lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, Q4_0, BF16 = 0, 1, 2, 30
EINVAL = -1


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        pytest.skip("libbrisk_hip.so is not built")
    return L.load()


# addresses that are never followed: every call here is refused or has nothing to do
AT = 1 << 20


def kv(**more):
    d = {"data": AT, "type": Q4_0, "kv_heads": 2, "head_dim": 64, "page_tokens": 16, "pages": 4, **more}
    return L.HipKv(**d)


def batch(**more):
    d = {"row_start": AT, "lengths": AT, "page_table": AT, "seqs": 2, "rows": 2, "page_stride": 4, "max_rows": 1, "max_length": 64, **more}
    return L.HipBatch(**d)


def heads(**more):
    return L.HipHeads(**{"data": AT, "type": F16, "row_stride": 128, "head_stride": 64, **more})


def rope(**more):
    return L.HipRope(**{"table": AT, "positions": 100, "dims": 64, "neox": 1, **more})


def r(x):
    return None if x is None else C.byref(x)


def refused(lib, rc, words):
    assert rc == EINVAL
    assert words in lib.brisk_hip_last_error().decode(), lib.brisk_hip_last_error()


def test_sizes(lib):
    # 16-bit rows take 2 bytes a value, 4-bit rows 18 bytes for 32
    for dim in (64, 96, 128, 256, 512):
        values = 2 * 3 * 32 * 10 * dim
        assert lib.brisk_hip_kv_bytes(r(kv(type=F16, kv_heads=3, head_dim=dim, page_tokens=32, pages=10))) == 2 * values
        assert lib.brisk_hip_kv_bytes(r(kv(type=Q4_0, kv_heads=3, head_dim=dim, page_tokens=32, pages=10))) == values * 18 // 32
    big = kv(type=F16, kv_heads=8, head_dim=128, page_tokens=64, pages=1 << 20)
    assert lib.brisk_hip_kv_bytes(r(big)) == (1 << 20) * 64 * 8 * 128 * 4


BAD_KV = [dict(type=F32), dict(type=8), dict(kv_heads=0), dict(kv_heads=2000), dict(head_dim=80), dict(head_dim=1024), dict(head_dim=0), dict(page_tokens=8),
          dict(page_tokens=48), dict(page_tokens=2048), dict(pages=0), dict(pages=1 << 31)]


@pytest.mark.parametrize("more", BAD_KV)
def test_cache_shapes_refused(lib, more):
    c = kv(**more)
    assert lib.brisk_hip_kv_bytes(r(c)) == 0
    assert lib.brisk_hip_paged_attention_bytes(r(c), r(batch()), 4) == 0
    b, h = batch(), heads()
    refused(lib, lib.brisk_hip_kv_append(r(c), r(b), r(h), r(h), None, 0.0, None, None), "a cache is F16 or Q4_0")
    refused(lib, lib.brisk_hip_kv_read(r(c), r(b), r(h), r(h), None), "a cache is F16 or Q4_0")
    refused(lib, lib.brisk_hip_paged_attention(r(c), r(b), r(h), 4, 1.0, 0, r(h), None, 0, None), "a cache is F16 or Q4_0")


def test_null_and_unaligned_arguments_refused(lib):
    h = heads()
    assert lib.brisk_hip_kv_bytes(None) == 0
    for c, b, words in [(None, batch(), "null cache"), (kv(data=None), batch(), "null cache"), (kv(data=AT + 8), batch(), "16-byte aligned"), (kv(), None, "null batch"),
                        (kv(), batch(row_start=None), "null row starts"), (kv(), batch(lengths=None), "null row starts"),
                        (kv(), batch(page_table=None), "null page table"), (kv(), batch(lengths=AT + 2), "not aligned"), (kv(), batch(rows=1 << 31), "too many rows")]:
        refused(lib, lib.brisk_hip_kv_append(r(c), r(b), r(h), r(h), None, 0.0, None, None), words)
        refused(lib, lib.brisk_hip_kv_read(r(c), r(b), r(h), r(h), None), words)
        refused(lib, lib.brisk_hip_paged_attention(r(c), r(b), r(h), 4, 1.0, 0, r(heads(row_stride=256)), AT, 1 << 30, None), words)


@pytest.mark.parametrize("x,words", [(None, "null"), (dict(data=None), "null"), (dict(type=Q4_0), "must be F32, F16 or BF16"), (dict(data=AT + 1), "not aligned to its type"),
                                     (dict(type=F32, data=AT + 2), "not aligned to its type"), (dict(row_stride=1 << 62), "stride")])
def test_rows_refused(lib, x, words):
    x, h, c, b = None if x is None else heads(**x), heads(), kv(), batch()
    refused(lib, lib.brisk_hip_kv_append(r(c), r(b), r(x), r(h), None, 0.0, None, None), words)
    refused(lib, lib.brisk_hip_kv_append(r(c), r(b), r(h), r(x), None, 0.0, None, None), words)
    if x is not None:
        refused(lib, lib.brisk_hip_kv_read(r(c), r(b), r(x), None, None), words)
    o = heads(row_stride=256)
    refused(lib, lib.brisk_hip_paged_attention(r(c), r(b), r(x), 4, 1.0, 0, r(o), AT, 1 << 30, None), words)
    refused(lib, lib.brisk_hip_paged_attention(r(c), r(b), r(o), 4, 1.0, 0, r(x), AT, 1 << 30, None), words)
    refused(lib, lib.brisk_hip_qk_norm_rope(r(x), None, 2, 2, 0, 64, None, None, 0.0, None, None, r(h), None, None), words)
    refused(lib, lib.brisk_hip_qk_norm_rope(r(h), None, 2, 2, 0, 64, None, None, 0.0, None, None, r(x), None, None), words)


@pytest.mark.parametrize("strides", [(0, 64), (64, 64), (128, 0), (128, 32), (127, 64), (64, 64 * 1)])
def test_outputs_that_overlap_refused(lib, strides):
    o = heads(row_stride=strides[0], head_stride=strides[1])
    refused(lib, lib.brisk_hip_kv_read(r(kv()), r(batch()), r(o), None, None), "overlap")
    refused(lib, lib.brisk_hip_qk_norm_rope(r(heads()), None, 2, 2, 0, 64, None, None, 0.0, None, None, r(o), None, None), "overlap")


@pytest.mark.parametrize("more,words", [(dict(table=None), "empty rotation"), (dict(positions=0), "empty rotation"), (dict(dims=0), "even and at most"), (dict(dims=7), "even and at most"),
                                        (dict(dims=66), "even and at most"), (dict(neox=0), "neox"), (dict(neox=3), "neox"), (dict(table=AT + 2), "aligned")])
def test_rotations_refused(lib, more, words):
    t, h = rope(**more), heads()
    refused(lib, lib.brisk_hip_kv_append(r(kv()), r(batch()), r(h), r(h), None, 0.0, r(t), None), words)
    refused(lib, lib.brisk_hip_qk_norm_rope(r(h), None, 2, 2, 0, 64, None, None, 0.0, r(t), AT, r(h), None, None), words)


def test_norm_rope_refusals(lib):
    h = heads()

    def call(q=h, k=None, n=2, nh=2, nk=2, dim=64, eps=0.0, t=None, pos=None, qo=h, ko=None):
        return lib.brisk_hip_qk_norm_rope(r(q), r(k), n, nh, nk, dim, None, None, eps, r(t), pos, r(qo), r(ko), None)

    refused(lib, call(dim=60), "multiple of 8")
    refused(lib, call(dim=520), "multiple of 8")
    refused(lib, call(dim=0), "multiple of 8")
    refused(lib, call(nh=0), "head count")
    refused(lib, call(k=h, ko=h, nk=0), "head count")
    refused(lib, call(k=h), "keys need an output")
    refused(lib, call(ko=h), "keys need an output")
    refused(lib, call(eps=-1.0), "eps")
    refused(lib, call(eps=float("nan")), "eps")
    refused(lib, call(t=rope()), "null positions")
    refused(lib, call(t=rope(), pos=AT + 2), "aligned")
    assert call(n=0, q=None, qo=None) == 0


def test_attention_refusals(lib):
    c, b, q = kv(), batch(), heads(row_stride=256)

    def call(heads_=4, scale=1.0, work=AT, size=1 << 30, b=b, c=c):
        return lib.brisk_hip_paged_attention(r(c), r(b), r(q), heads_, scale, 0, r(q), work, size, None)

    refused(lib, call(heads_=0), "multiple of the key/value heads")
    refused(lib, call(heads_=3), "multiple of the key/value heads")
    refused(lib, call(scale=float("inf")), "finite")
    refused(lib, call(scale=float("nan")), "finite")
    refused(lib, call(heads_=65536, b=batch(rows=1 << 20)), "too many rows and heads")
    long = batch(page_stride=4096, max_length=60000)
    need = lib.brisk_hip_paged_attention_bytes(r(c), r(long), 4)
    assert need > 0
    refused(lib, call(b=long, size=need - 1), f"needs {need} bytes")
    refused(lib, call(b=long, work=None, size=need), f"needs {need} bytes")
    refused(lib, call(b=long, work=AT + 4, size=need), "16-byte aligned")
    assert lib.brisk_hip_paged_attention_bytes(r(c), r(long), 3) == 0
    assert lib.brisk_hip_paged_attention_bytes(r(c), None, 4) == 0


def test_nothing_to_do(lib):
    for b in (batch(rows=0), batch(seqs=0, row_start=None, lengths=None, page_table=None)):
        assert lib.brisk_hip_kv_append(r(kv()), r(b), None, None, None, 0.0, None, None) == 0
        assert lib.brisk_hip_kv_read(r(kv()), r(b), None, None, None) == 0
        assert lib.brisk_hip_paged_attention(r(kv()), r(b), None, 4, 1.0, 0, None, None, 0, None) == 0
        assert lib.brisk_hip_paged_attention_bytes(r(kv()), r(b), 4) == 0
    assert lib.brisk_hip_kv_read(r(kv()), r(batch()), None, None, None) == 0


PROBE = r'''
#include <cstdio>
#include <cstring>
#include <vector>
#include "paged.h"
using namespace bh;
static int bad(const char* what, long a, long b) { std::printf("%s %ld %ld\n", what, a, b); return 1; }
int main() {
    // every byte of a tile belongs to one value, scale or code, and none lies outside
    for (int q4 = 0; q4 < 2; ++q4)
        for (uint32_t nb : {2u, 3u, 4u, 8u, 16u}) {
            std::vector<int> n(tile_bytes(q4, nb), 0);
            for (uint32_t t = 0; t < 16; ++t)
                for (uint32_t d = 0; d < 32 * nb; d += 2) {
                    const uint32_t o = value_offset(q4, nb, t, d);
                    for (int j = 0; j < (q4 ? 1 : 4); ++j) { if (o + j >= n.size()) return bad("value", nb, o); ++n[o + j]; }
                    if (d % 8 == 0) {
                        const uint32_t k = key_offset(q4, nb, t, d);
                        if (k % (q4 ? 4 : 16)) return bad("alignment", nb, k);
                        for (int j = 0; j < (q4 ? 4 : 16); ++j) { if (k + j >= n.size()) return bad("key", nb, k); ++n[k + j]; }
                    }
                    if (q4 && d % 32 == 0)
                        for (int v = 0; v < 2; ++v)
                            for (int j = 0; j < 2; ++j) { const uint32_t s = scale_offset(nb, v, t, d / 32) + j; if (s >= n.size()) return bad("scale", nb, s); ++n[s]; }
                }
            for (size_t j = 0; j < n.size(); ++j) if (n[j] != 1) return bad("count", nb, (long)j);
        }
    // pages: tables' ends, entries that are no page, positions before 0
    int32_t table[8] = {3, -1, 9, 0, 10, 2147483647, -2147483647, 1}, starts[5] = {0, 4, 2, 9, 40}, lengths[4] = {70, 5, -3, 100};
    PagedKv kv{nullptr, 1, 2, 64, 32, 10, 5};
    PagedBatch b{starts, lengths, table, 4, 20, 4, 0, 0};
    const long want[][3] = {{0, 0, 3}, {0, 31, 3}, {0, 32, -1}, {0, 64, 9}, {0, 127, 0}, {0, 128, -1}, {0, -1, -1}, {1, 0, -1}, {1, 32, -1}, {1, 64, -1}, {1, 96, 1}, {1, 0x7FFFFFFF, -1}};
    for (auto& w : want) if (page_of(kv, b, (uint32_t)w[0], (int32_t)w[1]) != w[2]) return bad("page", w[0], w[1]);
    // a page's tiles follow each other and end with the cache
    if (tile_at(kv, 9, 1, 31) + tile_bytes(true, 2) != size_t(10) * 2 * 2 * tile_bytes(true, 2)) return bad("end", 0, 0);
    if (tile_at(kv, 0, 0, 15) != 0 || tile_at(kv, 0, 0, 16) != tile_bytes(true, 2) || tile_at(kv, 0, 1, 0) != 2 * tile_bytes(true, 2)) return bad("order", 0, 0);
    PagedKv big{nullptr, 0, 8, 128, 64, 1u << 20, 6};
    if (tile_at(big, (1 << 20) - 1, 7, 63) + tile_bytes(false, 4) != (size_t(1) << 20) * 8 * 4 * tile_bytes(false, 4)) return bad("64 bits", 0, 0);
    // rows: never outside the tensors, whatever the starts say
    SeqRows r = seq_rows(b, 0);
    if (r.begin != 0 || r.end != 4 || r.first != 66) return bad("rows", 0, r.first);
    r = seq_rows(b, 1);
    if (r.begin != r.end) return bad("rows", 1, r.end);
    r = seq_rows(b, 2);
    if (r.begin != 2 || r.end != 9 || r.first != -7) return bad("rows", 2, r.first);
    r = seq_rows(b, 3);
    if (r.begin != 9 || r.end != 20 || r.first != 69) return bad("rows", 3, r.first);
    for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 8u, 20u, 96u, 641u, 1024u, 65535u, 65536u}) {
        const Divisor v = divisor(d);
        for (uint32_t n : {0u, 1u, d - 1, d, d + 1, 7 * d - 1, 7 * d, 0x7FFFFFFFu / d * d - 1, 0x7FFFFFFFu / d * d, 0x7FFFFFFEu, 0x7FFFFFFFu})
            if (over(n & 0x7FFFFFFF, v) != (n & 0x7FFFFFFF) / d) return bad("division", d, n);
    }
    starts[1] = 2147483647; lengths[0] = 2147483647;
    r = seq_rows(b, 0);
    if (r.begin != 0 || r.end != 20 || r.first != kMaxLength - 2147483647) return bad("rows", 5, r.first);
    starts[1] = 4; lengths[0] = 70;
    starts[0] = -5;
    r = seq_rows(b, 0);
    if (r.begin != 0 || r.end != 4 || r.first != 66) return bad("rows", 4, r.first);
    return 0;
}
'''


def test_places_on_the_host(tmp_path):
    """csrc/paged.h's functions, as the kernels use them, compiled for the host."""
    src, exe = tmp_path / "places.cpp", tmp_path / "places"
    src.write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(ROOT, "brisk-llm_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


def test_reference_rows_by_hand():
    """The tests' own plain form: a block by hand."""
    import paged_reference as R
    x = np.zeros((1, 32))
    x[0, :4] = [8, -8, 7.4, 0.5]
    v, near = R.held(x, Q4_0)
    assert v[0, :4].tolist() == [8, -7, 7, 0] or v[0, 0] == 8
    # d = -1: codes floor(-x + 8.5) = 0, 16 -> 15, floor(1.1) = 1, floor(8.0) = 8
    assert v[0, :4].tolist() == [8.0, -7.0, 7.0, 0.0]
