"""The module that puts the operators on torch tensors: it loads without a GPU, on top of the library that is loaded, or says why not."""

from __future__ import annotations

import pytest

from spear_b200 import _lib


def test_loads_once_and_names_its_functions():
    module = _lib.native()
    assert module is _lib.native()
    assert {"rms_norm", "causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step"} <= set(dir(module))
    with open("/proc/self/maps") as maps:  # one copy of the library, whoever asked for it
        assert len({line.split()[-1] for line in maps if "libbtp_sm100" in line}) == 1


def test_says_why_it_does_not_load(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_module", None)
    monkeypatch.setattr(_lib, "MODULE_PATH", str(tmp_path / "btp_torch.so"))
    with pytest.raises(_lib.BtpLibraryError, match="missing"):
        _lib.native()
    (tmp_path / "btp_torch.so").write_bytes(b"no library")
    with pytest.raises(_lib.BtpLibraryError, match="does not load"):
        _lib.native()
