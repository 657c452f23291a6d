"""CPU checks of the serving operators: the cache's layout and which rows, pages and keys a batch's
arrays name (cache_layout.h, whatever the arrays hold), and the calls that are refused before any
device work."""

import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fusor-ai_amd", "csrc")
SOURCE = """
#include "cache_layout.h"
using namespace fg;
extern "C" {
int padded(int d) { return padded_head(d); }
int bytes(int p) { return record_bytes(p); }
int kbyte(int p, int t, int d) { return key_byte(p, t, d); }
int vbyte(int p, int t, int d) { return value_byte(p, t, d); }
int kscale(int p, int t) { return key_scale_byte(p, t); }
int vscale(int p, int t) { return value_scale_byte(p, t); }
void span(int a, int b, int n, int total, int *out)
{ Span s = span_of(a, b, n, total); out[0] = s.begin; out[1] = s.rows; out[2] = s.first; out[3] = s.length; }
int page(const int32_t *t, int i, int columns, int pages) { return page_at(t, i, columns, pages); }
void seen(int a, int b, int n, int total, int row, int last, int window, int columns, int *out)
{ PageRange r = pages_seen(span_of(a, b, n, total), row, last, window, columns); out[0] = r.lo; out[1] = r.hi; }
void news(int a, int b, int n, int total, int *out)
{ PageRange r = pages_of_new(span_of(a, b, n, total)); out[0] = r.lo; out[1] = r.hi; }
}
"""


@pytest.fixture(scope="module")
def layout(tmp_path_factory):
    where = tmp_path_factory.mktemp("layout")
    source, lib = where / "layout.cpp", where / "layout.so"
    source.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC,
                    str(source), "-o", str(lib)], check=True)
    return ctypes.CDLL(str(lib))


@pytest.mark.parametrize("dim", [4, 32, 36, 64, 72, 96, 128, 132, 192, 256])
def test_a_record_holds_every_level_once(layout, dim):
    padded = layout.padded(dim)
    assert padded >= dim and padded in (32, 64, 96, 128, 192, 256)
    keys = [layout.kbyte(padded, t, d) for t in range(64) for d in range(padded)]
    values = [layout.vbyte(padded, t, d) for t in range(64) for d in range(padded)]
    scales = [layout.kscale(padded, t) for t in range(64)] + [layout.vscale(padded, t) for t in range(64)]
    assert sorted(keys) == list(range(64 * padded))
    assert sorted(values) == list(range(64 * padded, 128 * padded))
    assert sorted(scales) == list(range(128 * padded, 128 * padded + 512, 4))
    assert layout.bytes(padded) == 128 * padded + 512
    # runs that the kernels move whole: four dimensions of a key, four tokens of a value, a value's scales
    for t in range(0, 64, 4):
        for d in range(0, dim, 4):
            assert [layout.kbyte(padded, t, d + i) - layout.kbyte(padded, t, d) for i in range(4)] == [0, 1, 2, 3]
            assert [layout.vbyte(padded, t + i, d) - layout.vbyte(padded, t, d) for i in range(4)] == [0, 1, 2, 3]


BIG = 2 ** 31 - 1
ARRAYS = [(0, 5, 9, 10), (0, 0, 7, 10), (3, 2, 7, 10), (-5, 4, 2, 10), (8, 99, 70, 10), (99, 120, 5, 10), (0, 10, -3, 10),
          (0, 10, BIG, 10), (BIG, -BIG - 1, BIG, 10), (0, 3, 0, 3), (0, 200, 130, 200), (0, 1, 1, 1), (0, 64, 64, 64),
          (0, 65, 128, 65)]


@pytest.mark.parametrize("arrays", ARRAYS)
def test_rows_and_pages_stay_inside_the_operands(layout, arrays):
    total = arrays[3]
    out = (ctypes.c_int * 4)()
    layout.span(*arrays, out)
    begin, rows, first, length = out
    assert 0 <= begin <= total and rows >= 0 and begin + rows <= total and length >= 0 and first == length - rows
    r = (ctypes.c_int * 2)()
    layout.news(*arrays, r)
    if rows:
        assert r[0] == first // 64 and r[1] == (first + rows - 1) // 64 + 1
        assert r[1] - r[0] <= (rows + 62) // 64 + 1
    else:
        assert r[0] == r[1]
    for columns in (0, 1, 2, 5, 1 << 24):
        for window in (0, 1, 63, 64, 65, 100000, BIG):
            for row in {0, rows // 2, rows - 1} if rows else ():
                for last in {row, rows - 1}:
                    layout.seen(*arrays, row, last, window, columns, r)
                    low = max(0, first + row - window + 1) if window else 0
                    high = first + last + 1  # keys low .. high - 1
                    assert 0 <= r[0] <= r[1] <= columns
                    if high > low:
                        assert r[0] == min(low // 64, r[1]) and r[1] == min((high - 1) // 64 + 1, columns)
                    elif high <= 0:
                        assert r[0] == r[1]


def test_page_ids_outside_the_cache_hold_nothing(layout):
    table = (ctypes.c_int32 * 4)(2, -1, 7, BIG)
    assert [layout.page(table, i, 4, 7) for i in (-1, 0, 1, 2, 3, 4)] == [-1, 2, -1, -1, -1, -1]
    assert layout.page(table, 2, 4, 8) == 7
    assert layout.page(None, 0, 0, 8) == -1  # no columns: the table is not read


def call(name, *args):
    from fusor_kernels import _lib
    rc = getattr(_lib.lib(), name)(*args)
    return rc, _lib.lib().fg_last_error().decode()


def test_refusals_before_any_device_work():
    from fusor_kernels import _lib
    handle = ctypes.c_void_p()
    for heads, dim in [(0, 64), (2, 0), (2, 62), (2, 260), (5000, 64)]:
        rc, message = call("fg_cache_create", 4, heads, dim, None, ctypes.byref(handle))
        assert rc == _lib.FG_ERR_SHAPE and "fg_cache_create" in message and not handle
    assert call("fg_cache_create", (1 << 24) + 1, 2, 64, None, ctypes.byref(handle))[0] == _lib.FG_ERR_SHAPE
    assert call("fg_cache_create", 4, 2, 64, None, None)[0] == _lib.FG_ERR_ARG
    batch = _lib.FgBatch(1, 1, 1, None, None, None)
    for rc, message in (call("fg_cache_write", None, ctypes.byref(batch), None, 0, None, 0, None),
                        call("fg_cache_read", None, ctypes.byref(batch), None, 0, None, 0, None),
                        call("fg_cache_attend", None, ctypes.byref(batch), None, 0, 2, 1.0, 0, None, 0, None, 0, None)):
        assert rc == _lib.FG_ERR_ARG and "null cache" in message
    settings = _lib.FgSampling(None, None, None, None, None)
    some = ctypes.c_void_p(256)  # refused before it is looked at
    assert call("fg_sample", some, 1, 8, 8, None, some, None, None, 0, None)[0] == _lib.FG_ERR_ARG
    assert call("fg_sample", some, 1, 8, 8, ctypes.byref(settings), some, None, None, 0, None)[0] == _lib.FG_ERR_ARG
    assert call("fg_sample", some, 1, 0, 8, ctypes.byref(settings), some, None, None, 0, None)[0] == _lib.FG_ERR_SHAPE
    assert call("fg_sample", some, 1, (1 << 22) + 1, 8, ctypes.byref(settings), some, None, None, 0, None)[0] == _lib.FG_ERR_SHAPE
    assert call("fg_sample", some, (1 << 20) + 1, 8, 8, ctypes.byref(settings), some, None, None, 0, None)[0] == _lib.FG_ERR_SHAPE
    assert call("fg_sample", None, 0, 8, 8, ctypes.byref(settings), None, None, None, 0, None)[0] == _lib.FG_OK  # no rows
    # scratch sizes: of calls that would be refused, none
    sizes = _lib.lib().fg_sample_scratch
    assert sizes(0, 8) == sizes(8, 0) == sizes(1, (1 << 22) + 1) == 0 and 0 < sizes(1, 8) <= sizes(7, 8) <= sizes(7, 151936)
    assert _lib.lib().fg_cache_attend_scratch(None, ctypes.byref(batch), 2) == 0


def test_the_plain_forms_agree_with_torch():
    """The tests' own 64-bit forms against torch's softmax and a whole draw by counting."""
    import numpy as np
    import torch
    import serving
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(5, n, 8, generator=g).double() for n in (4, 2, 2))
    mask = torch.tril(torch.ones(5, 5, dtype=torch.bool))
    want = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(0, 1), k.repeat_interleave(2, 1).transpose(0, 1), v.repeat_interleave(2, 1).transpose(0, 1), mask)
    got = serving.attention(q, k, v, range(5), 8 ** -0.5)[0]
    assert torch.allclose(got, want.transpose(0, 1), rtol=1e-12, atol=1e-13)
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    draws = [serving.draw(x, u)[0] for u in (0.0, 0.099, 0.101, 0.499, 0.501, 0.699, 0.701, 0.999)]
    assert draws == [0, 0, 1, 1, 2, 2, 3, 3]
    assert serving.draw(x, 0.5, top_k=2) == (1, pytest.approx(4 / 7)) and serving.draw(x, 0.6, top_p=0.65)[0] == 3
    assert serving.draw(x, 0.0, min_p=0.5)[0] == 1 and serving.draw(x, 0.9, temperature=0.0) == (1, 1.0)
