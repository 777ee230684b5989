"""The extension module and the kernel library share records that two builds know: what keeps them together."""
import ctypes
import importlib.util

import pytest
import torch

from torsh_b200 import _build, _native as nv

NAMES = ("tb_set_device", "tb_last_error", "tb_rotary", "tb_kv_write", "tb_kv_read", "tb_cache_attention", "tb_cache_attention_workspace", "tb_verify_draft",
         "tb_decode_layout")


def _module():
    path = _build.build_torch()
    spec = importlib.util.spec_from_file_location("torsh_b200._decode_calls", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_a_library_of_other_records_is_refused():
    import sys
    _build.build_cuda()
    lib, mod = nv.cuda(), _module()
    lib.tb_decode_layout.restype = ctypes.c_uint64
    assert hex(lib.tb_decode_layout()) == _build._decode_layout().split("=")[1].replace("0x0", "0x")
    other = ctypes.CFUNCTYPE(ctypes.c_uint64)(lambda: 1)
    address = lambda f: ctypes.c_void_p.from_address(ctypes.addressof(f)).value   # noqa: E731
    good = [address(getattr(lib, n)) for n in NAMES]
    with pytest.raises(nv.NativeError, match="different records"):
        mod.bind(sys.modules[nv.__name__], *good[:-1], address(other))
    for bad in (good[:-1], good + [1]):
        with pytest.raises(TypeError):
            mod.bind(sys.modules[nv.__name__], *bad)
    with pytest.raises(ValueError):
        mod.bind(sys.modules[nv.__name__], *good[:-1], 0)
    mod.bind(sys.modules[nv.__name__], *good)
    assert mod.torch_version == torch.__version__.split("+")[0]


def test_the_module_is_built_again_for_another_pytorch(monkeypatch, tmp_path):
    """Nothing is compiled here: what counts is that the build would be."""
    _build.build_torch()
    made = []
    monkeypatch.setattr(_build, "OBJDIR", tmp_path)
    monkeypatch.setattr(_build, "_run", lambda cmd, verbose: made.append(cmd))
    _build.build_torch()
    assert len(made) == 1
    _build.build_torch()
    assert len(made) == 1                                                   # up to date
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    _build.build_torch()
    assert len(made) == 2
