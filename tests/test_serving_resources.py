"""What the compiler gave the serving kernels, by the metadata of the built library: none of them keeps a vector register, or
an array, in scratch memory. (A form of the row sampler that kept 127 there drew wrong tokens; other flags than the
Makefile's make the attention of wide heads spill.)"""

import os
import re
import shutil
import struct
import subprocess

import pytest

from fusor_kernels import _lib

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
READELF = shutil.which("llvm-readelf") or "/opt/rocm/llvm/bin/llvm-readelf"
KERNELS = {"cache_clear_kernel": 1, "cache_rows_kernel": 2, "cache_pages_kernel": 2, "attend_few_kernel": 6, "attend_many_kernel": 6,
           "attend_join_kernel": 12, "sample_top_kernel": 1, "sample_bins_kernel": 1, "sample_cut_kernel": 1,
           "sample_collect_kernel": 1, "sample_draw_kernel": 1, "sample_row_kernel": 1}


def code_objects(library):
    """The gfx950 code objects of a library: one bundle a source file, entries of (offset, size, length of name, name)."""
    at = library.find(MAGIC)
    while at >= 0:
        (count,) = struct.unpack_from("<Q", library, at + len(MAGIC))
        place = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", library, place)
            name = library[place + 24:place + 24 + length]
            place += 24 + length
            if b"gfx950" in name and size:
                yield library[at + offset:at + offset + size]
        at = library.find(MAGIC, at + 1)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    where = tmp_path_factory.mktemp("code") / "object"
    with open(_lib.LIB_PATH, "rb") as f:
        library = f.read()
    found = {}
    for code in code_objects(library):
        where.write_bytes(code)
        notes = subprocess.run([READELF, "--notes", str(where)], check=True, capture_output=True, text=True).stdout
        for kernel in re.split(r"\n  - ", notes)[1:]:  # each starts with its first field
            fields = dict(re.findall(r"^ *\.(name|private_segment_fixed_size|vgpr_spill_count): +(\S+)$", kernel, re.M))
            if "vgpr_spill_count" in fields:
                found[fields["name"].strip("'")] = fields
    return found


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
@pytest.mark.parametrize("name", sorted(KERNELS))
def test_no_scratch_memory(kernels, name):
    of = {symbol: fields for symbol, fields in kernels.items() if name in symbol}
    assert len(of) == KERNELS[name], sorted(kernels)
    for symbol, fields in of.items():
        assert int(fields["vgpr_spill_count"]) == 0 and int(fields["private_segment_fixed_size"]) == 0, (symbol, fields)
