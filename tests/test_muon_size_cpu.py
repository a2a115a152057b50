"""The size of Muon's step stands in one place."""
import ctypes
import pathlib
import re

import torch

from zorse_b200.ops import muon
from zorse_b200.ops import sm100 as k


def test_the_kernels_are_handed_the_size(monkeypatch):
    seen = {}

    class Lib:
        def zb_newton_schulz_workspace(self, table, count, limit, at):
            ctypes.c_long.from_address(at).value = 16
            return 0

        def zb_newton_schulz(self, *args):
            seen["args"] = args
            return 0

    monkeypatch.setattr(k, "_lib", Lib())
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)
    monkeypatch.setattr(k, "_stream", lambda: None)
    monkeypatch.setattr(k, "status_word", lambda dev: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(k, "_workspace_size", lambda *a: 16)
    u = torch.ones(3, 4)
    k.muon_step([u.clone()], [u.clone()], [u.clone()], [None], lr=0.5)
    assert (*muon.COEFFICIENTS, muon.SCALE) == k.NEWTON_SCHULZ and seen["args"][9:13] == k.NEWTON_SCHULZ
    text = (pathlib.Path(k.__file__).resolve().parents[2] / "csrc/optim/newton_schulz.cu").read_text()
    assert not re.search(r"\b0\.2f?\b", re.sub(r"//[^\n]*", "", text))
