"""CPU checks of the calls over shared prefixes: what is refused before any device work."""

import ctypes

import pytest


def test_refusals_before_any_device_work():
    from fusor_kernels import _lib
    lib = _lib.lib()
    batch, prefixes, some = _lib.FgBatch(1, 1, 1, None, None, None), _lib.FgPrefixes(1, 256, 256), ctypes.c_void_p(256)

    def call(cache, prefixes):
        return lib.fg_cache_attend_shared(cache, ctypes.byref(batch), prefixes, some, 0, 2, 1.0, 0, some, 0, None, 0, None)

    assert call(None, ctypes.byref(prefixes)) == _lib.FG_ERR_ARG and "null cache" in lib.fg_last_error().decode()
    assert call(None, None) == _lib.FG_ERR_ARG and "null prefixes" in lib.fg_last_error().decode()
    for bad, code in ((_lib.FgPrefixes(65537, 256, 256), _lib.FG_ERR_SHAPE), (_lib.FgPrefixes(1, None, 256), _lib.FG_ERR_ARG),
                      (_lib.FgPrefixes(1, 256, None), _lib.FG_ERR_ARG)):
        assert call(None, ctypes.byref(bad)) == code
    size = lib.fg_cache_attend_shared_scratch
    assert size(None, ctypes.byref(batch), ctypes.byref(prefixes), 2) == 0


def test_prefixes_are_device_tensors():
    import torch
    import fusor_kernels as fk
    starts, pages = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(fk.ShapeError, match="device tensor"):
        fk.Prefixes(starts, pages)
    with pytest.raises(fk.ShapeError):
        fk.Prefixes(starts, pages.view(1, 1))
