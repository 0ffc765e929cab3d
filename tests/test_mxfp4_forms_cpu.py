"""The forms of the 4-bit experts' backward that the library holds are those that its rules choose (CPU only)."""

from __future__ import annotations

import re

import pytest

from moe_mi355 import _lib

pytestmark = pytest.mark.cpu


def test_every_backward_form_is_reached():
    """The product with Wd (dact) has tiles of 64 or 128 rows, the one with the gate and up weights (dxp) of 256 too."""
    with open(_lib.LIB_PATH, "rb") as f:
        lib = f.read()
    for kernel in (b"k_mx_back", b"k_mx_back_reduce"):
        name = rb"\d%sINS0_6BkFormILi(\d)ELi(\d)ELi(\d)ELi(\d)ELi(\d)EEELb([01])EEEv" % kernel
        forms = {tuple(int(v) for v in m) for m in re.findall(name, lib)}
        rows = {(32 * tf * wt, bool(dact)) for tf, _nf, wt, _wf, _ks, dact in forms}
        assert rows == {(64, True), (128, True), (64, False), (128, False), (256, False)}, (kernel, forms)
