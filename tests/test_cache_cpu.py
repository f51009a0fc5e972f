"""The MXFP8 cache without a GPU: its index arithmetic, bad indexes among it,
compiled from the kernels' own header; the binding; what is refused before a
device is touched."""

import ctypes
import pathlib
import re
import subprocess

import numpy as np
import pytest
import torch

import MXFP8_quantizer

ROOT = pathlib.Path(__file__).resolve().parent.parent
pkg = MXFP8_quantizer.load_package()
capi = pkg._capi


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    out = tmp_path_factory.mktemp("probe") / "cache_index.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-o", str(out), str(ROOT / "tests" / "cache_index_probe.cpp")], check=True)
    lib = ctypes.CDLL(str(out))
    i64, i32, vp = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p
    for name, args in (("probe_row", [i64, i32, i32, i64, i32, i32]), ("probe_table", [vp, i64, i64, i64, i64, i32]),
                       ("probe_sequence", [vp, i64, i64, i64]), ("probe_begin", [i64] * 3), ("probe_part", [i64] * 3),
                       ("probe_visible", [i64, i64, i32])):
        getattr(lib, name).argtypes, getattr(lib, name).restype = args, i64
    return lib


def test_rows_stay_inside_the_cache(probe):
    pages, heads, shift = 7, 3, 4
    seen = set()
    for page in range(pages):
        for head in range(heads):
            for offset in range(16):
                row = probe.probe_row(pages, heads, shift, page, head, offset)
                assert row == (page * heads + head) * 16 + offset
                seen.add(row)
    assert seen == set(range(pages * heads * 16))
    for bad in (-1, -2 ** 31, pages, 2 ** 31 - 1, 2 ** 40):
        assert probe.probe_row(pages, heads, shift, bad, 0, 0) == -1
    # past 32 bits: the last row of 2^32 - 64
    assert probe.probe_row((2 ** 32 - 64) // 32, 2, 4, (2 ** 32 - 64) // 32 - 1, 1, 15) == 2 ** 32 - 65


def test_positions_past_the_table_have_no_page(probe):
    table = np.array([[4, -1, 99], [5, 6, 2 ** 31 - 1]], np.int32)
    at = lambda b, i: probe.probe_table(table.ctypes.data, 3, 3, b, i, 3)  # noqa: E731
    assert [at(0, 0), at(0, 7), at(0, 8), at(0, 16), at(1, 0), at(1, 23)] == [4, 4, -1, 99, 5, 2 ** 31 - 1]
    assert at(0, 24) == -1 and at(1, 24) == -1 and at(0, 2 ** 40) == -1 and at(0, -1) == -1
    assert probe.probe_table(None, 0, 0, 0, 0, 3) == -1


@pytest.mark.parametrize("starts", [[0, 5], [0, 0, 0, 3, 3, 10, 10], [4, 4, 9], [0, 0], [2, 7, 7, 7, 8]])
def test_sequence_of_every_row(probe, starts):
    a = np.array(starts, np.int32)
    batch = len(starts) - 1
    for first, row in ((f, r) for r in range(-1, starts[-1] + 3) for f in range(max(-1, r - 4), r + 1)):
        got = probe.probe_sequence(a.ctypes.data, batch, first, row)
        if row < starts[0]:
            assert got == -1
        elif row >= starts[-1]:
            assert got == batch
        else:
            assert starts[got] <= row < starts[got + 1]


def test_sequence_of_falling_starts_stays_in_range(probe):
    """starts that fall break the contract; the answer still names a sequence, or none."""
    rng = np.random.default_rng(0)
    for _ in range(200):
        a = rng.integers(-5, 20, rng.integers(2, 9)).astype(np.int32)
        for row in range(-3, 22):
            assert -1 <= probe.probe_sequence(a.ctypes.data, len(a) - 1, row - 2, row) <= len(a) - 1


@pytest.mark.parametrize("n,total", [(1, 1), (1, 9), (3, 3), (3, 10), (7, 8), (444, 445), (444, 100000),
                                     (444, 3 * 2 ** 33 + 1)])
def test_split_covers_every_tile_once(probe, n, total):
    begins = [probe.probe_begin(i, n, total) for i in range(n + 1)]
    assert begins[0] == 0 and begins[-1] == total and all(a < b for a, b in zip(begins, begins[1:]))
    for i in range(n):
        for x in {begins[i], begins[i + 1] - 1, (begins[i] + begins[i + 1]) // 2}:
            assert probe.probe_part(x, n, total) == i


def test_visible_length(probe):
    for length, want in ((-5, 0), (0, 0), (1, 1), (48, 48), (49, 48), (2 ** 31 - 1, 48)):
        assert probe.probe_visible(length, 3, 4) == want


def test_header_binding_and_libraries_agree():
    text = (ROOT / "include" / "mxfp8_cache.h").read_text()
    declared = sorted(set(re.findall(r"MXFP8_API\s+[\w\s\*]+?\b(mxfp8_\w+)\s*\(", text)))
    assert declared == sorted(capi.CACHE_EXPORTS)
    for name in declared:
        assert hasattr(capi.lib(), name) and hasattr(capi.checked_lib(), name), name
    assert capi.strerror(capi.ERR_WORKSPACE) != "unknown status"


def a_cache(**change):
    a = dict(k=0x1000, v=0x2000, k_scales=0x3000, v_scales=0x4000, num_pages=4, heads=2, page_size=16, dim=128)
    a.update(change)
    return capi.Cache(*a.values())


BAD_CACHES = [(dict(k=0), "NULL"), (dict(v_scales=0), "NULL"), (dict(k=0x1008), "alignment"),
              (dict(k_scales=0x3002), "alignment"), (dict(num_pages=-1), "sizes"), (dict(heads=0), "sizes"),
              (dict(page_size=12), "sizes"), (dict(page_size=0), "sizes"), (dict(page_size=8192), "sizes"),
              (dict(dim=48), "sizes"), (dict(dim=0), "sizes"), (dict(dim=2048), "sizes"),
              (dict(num_pages=2 ** 28), "sizes")]


def write(cache, **change):
    a = dict(k=0x5000, kt=256, kh=128, v=0x6000, vt=256, vh=128, dtype=0, tokens=4, slots=0x7000, stream=0)
    a.update(change)
    capi.cache_write(cache, *a.values())


def read(cache, **change):
    a = dict(table=0x5000, stride=4, max_pages=4, batch=2, starts=0x6000, total=8, k=0x7000, v=0x8000, dtype=0, stream=0)
    a.update(change)
    capi.cache_read(cache, *a.values())


def attend(cache, **change):
    a = dict(q=0x5000, qb=512, qh=128, dtype=0, batch=2, heads=4, table=0x6000, stride=4, max_pages=4, lengths=0x7000,
             scale=1.0, out=0x8000, lse=0, ws=0x9000, ws_bytes=1 << 30, stream=0)
    a.update(change)
    capi.cache_attention(cache, *a.values())


@pytest.mark.parametrize("call", [write, read, attend])
@pytest.mark.parametrize("change,match", BAD_CACHES)
def test_bad_caches_are_refused(call, change, match):
    with pytest.raises(ValueError, match=match):
        call(a_cache(**change))


@pytest.mark.parametrize("heads", [65537, 2 ** 25, 2 ** 28, 2 ** 31 - 1])
@pytest.mark.parametrize("call", [write, read, attend])
def test_more_heads_than_32_bits_count_are_refused(call, heads):
    """Rows of a token: heads * dim / 16 of them a thread each; 2^28 heads of 128 elements are 2^32 eighths."""
    for pages in (0, 1):
        with pytest.raises(ValueError, match="sizes"):
            call(a_cache(num_pages=pages, page_size=2, heads=heads))


@pytest.mark.parametrize("call,change,match", [
    (write, dict(dtype=2), "dtype"), (write, dict(tokens=-1), "sizes"), (write, dict(kt=-1), "sizes"),
    (write, dict(k=0), "NULL"), (write, dict(slots=0), "NULL"), (write, dict(v=0x6001), "alignment"),
    (write, dict(slots=0x7004), "alignment"), (write, dict(tokens=2 ** 31), "sizes"),
    (read, dict(dtype=3), "dtype"), (read, dict(batch=-1), "sizes"), (read, dict(total=-1), "sizes"),
    (read, dict(total=2 ** 31), "sizes"), (read, dict(max_pages=-1), "sizes"), (read, dict(stride=-1), "sizes"),
    (read, dict(table=0), "NULL"), (read, dict(starts=0), "NULL"), (read, dict(k=0), "NULL"),
    (read, dict(v=0x8008), "alignment"),
    (attend, dict(dtype=2), "dtype"), (attend, dict(heads=3), "sizes"), (attend, dict(heads=0), "sizes"),
    (attend, dict(batch=-1), "sizes"), (attend, dict(max_pages=2 ** 28), "sizes"), (attend, dict(qh=-1), "sizes"),
    (attend, dict(q=0), "NULL"), (attend, dict(lengths=0), "NULL"), (attend, dict(out=0), "NULL"),
    (attend, dict(ws=0), "NULL"), (attend, dict(q=0x5001), "alignment"), (attend, dict(out=0x8008), "alignment"),
    (attend, dict(lse=0xA002), "alignment"), (attend, dict(ws=0x9008), "alignment"),
])
def test_bad_arguments_are_refused(call, change, match):
    with pytest.raises(ValueError, match=match):
        call(a_cache(), **change)


@pytest.mark.parametrize("change", [dict(dim=96), dict(dim=32), dict(page_size=1), dict(dim=512)])
def test_attention_refuses_geometries_it_has_no_kernel_for(change):
    with pytest.raises(ValueError, match="sizes"):
        attend(a_cache(**change))


def test_empty_calls_are_no_ops():
    empty = a_cache(k=0, v=0, k_scales=0, v_scales=0, num_pages=0)
    write(empty, tokens=0, k=0, v=0, slots=0)
    read(empty, batch=0, total=0)
    read(empty, total=0)
    attend(empty, batch=0)


def test_wrappers_refuse_wrong_tensors():
    cache = pkg.allocate_cache(4, 16, 2, 64, device="cpu")
    k = torch.zeros((5, 2, 64), dtype=torch.bfloat16)
    slots = torch.arange(5)
    table, lengths = torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    starts = torch.zeros(4, dtype=torch.int32)
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16)
    for call, match in (
            (lambda: pkg.cache_write(cache, k, k, slots), "CUDA"),
            (lambda: pkg.cache_write(cache, k[:, :1], k, slots), "k must"),
            (lambda: pkg.cache_write(cache, k, k[:4], slots), "same number"),
            (lambda: pkg.cache_write(cache, k, k.half(), slots), "one type"),
            (lambda: pkg.cache_write(cache, k.float(), k.float(), slots), "bfloat16"),
            (lambda: pkg.cache_write(cache, k, k, slots.int()), "int64"),
            (lambda: pkg.cache_write(cache._replace(v=cache.v[:3]), k, k, slots), "k and v must"),
            (lambda: pkg.cache_write(cache._replace(k=cache.k.transpose(1, 2), v=cache.v.transpose(1, 2)), k, k, slots),
             "scales must"),
            (lambda: pkg.cache_write(cache._replace(k_scales=cache.k_scales.float()), k, k, slots), "bytes"),
            (lambda: pkg.cache_read(cache, table, starts, 8), "CUDA"),
            (lambda: pkg.cache_read(cache, table.long(), starts, 8), "int32"),
            (lambda: pkg.cache_read(cache, table, starts[:3], 8), "batch"),
            (lambda: pkg.cache_read(cache, table, starts, -1), "total"),
            (lambda: pkg.cache_read(cache, table, starts, 8, torch.float64), "out_dtype"),
            (lambda: pkg.cache_read(cache, table, starts, 8, out=(k, k)), "out must"),
            (lambda: pkg.cache_attention(q, cache, table, lengths), "CUDA"),
            (lambda: pkg.cache_attention(q[:2], cache, table, lengths), "batch"),
            (lambda: pkg.cache_attention(q[:, :3], cache, table, lengths), "multiple"),
            (lambda: pkg.cache_attention(q.float(), cache, table, lengths), "bfloat16"),
            (lambda: pkg.cache_attention(q[:, :, :32], cache, table, lengths), "q must"),
            (lambda: pkg.cache_attention(q, cache, table, lengths.long()), "int32"),
            (lambda: pkg.cache_attention(q[:, :, :32], pkg.allocate_cache(4, 16, 2, 32, device="cpu"), table, lengths),
             "attention needs"),
    ):
        with pytest.raises(ValueError, match=match):
            call()
    for bad in ((4, 12, 2, 64), (4, 16, 0, 64), (4, 16, 2, 40), (-1, 16, 2, 64)):
        with pytest.raises(ValueError, match="a cache needs"):
            pkg.allocate_cache(*bad, device="cpu")
