"""Which of fg_sample's two forms a call takes (sample_route.h): for sizes measured more than a tenth
apart, the faster; and chunks that cover a row."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fusor-ai_amd", "csrc")

# rows, vocabulary, microseconds by rows and by chunks
MEASURED = [
    (16, 5000, 18, 28), (64, 5000, 17, 30), (256, 5000, 17, 33), (512, 5000, 30, 48), (64, 32003, 31, 37), (96, 32003, 29, 43),
    (200, 32003, 34, 53), (384, 32003, 60, 83), (512, 32003, 65, 88), (1, 151936, 74, 32), (16, 151936, 82, 41),
    (32, 151936, 81, 49), (64, 151936, 91, 65), (256, 151936, 106, 119), (384, 151936, 176, 213), (512, 151936, 199, 255),
]


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    where = tmp_path_factory.mktemp("route")
    source, lib = where / "route.cpp", where / "route.so"
    source.write_text('#include "sample_route.h"\n'
                      'extern "C" int by_rows(size_t rows, size_t vocab) { return fg::sample_by_rows(rows, vocab); }\n'
                      'extern "C" int chunks(size_t rows, size_t vocab, int by) { return fg::sample_chunks(rows, vocab, by != 0); }\n'
                      'extern "C" int chunk(size_t vocab, int by, int *chunks) { return fg::sample_chunk(vocab, by != 0, chunks); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(source), "-o", str(lib)], check=True)
    lib = ctypes.CDLL(str(lib))
    lib.by_rows.argtypes = [ctypes.c_size_t] * 2
    lib.chunks.argtypes = [ctypes.c_size_t] * 2 + [ctypes.c_int]
    lib.chunk.argtypes = [ctypes.c_size_t, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    return lib


@pytest.mark.parametrize("call", MEASURED)
def test_the_faster_form(route, call):
    rows, vocab, by_rows, by_chunks = call
    assert bool(route.by_rows(rows, vocab)) == (by_rows < by_chunks)


@pytest.mark.parametrize("vocab", [1, 4095, 4096, 8191, 32003, 151936, 1 << 22])
@pytest.mark.parametrize("rows", [1, 7, 64, 331, 2048])
def test_chunks(route, rows, vocab):
    for by in (0, 1):
        chunks = route.chunks(rows, vocab, by)
        assert 1 <= chunks <= 16
        left = ctypes.c_int(chunks)
        chunk = route.chunk(vocab, by, ctypes.byref(left))
        assert chunk % (4096 if by else 256) == 0 and 1 <= left.value <= chunks
        assert chunk * left.value >= vocab > chunk * (left.value - 1)  # no chunk is empty
