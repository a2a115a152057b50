"""Head norms: sizes that the kernels were not written for are refused by every entry point, the size of the workspace among them."""
import ctypes
import subprocess
import sys
import textwrap

import pytest
import torch

from zorse_b200.ops import sm100 as k

# run in a process of their own: a call that ends its process fails one test and not the run
WORKSPACE = """
    import ctypes
    from zorse_b200.ops import sm100 as k
    floats = ctypes.c_long(-1)
    rc = k.lib().zb_qk_norm_rope_workspace({T}, {nq}, {nk}, {d}, ctypes.addressof(floats))
    print(rc, floats.value, k.lib().zb_last_error().decode() if rc else "")
"""
BACKWARD = """
    import torch
    from zorse_b200.ops import sm100 as k
    k._bf16 = k._on_current = lambda t, name: None
    T, nq, nk, d = {T}, {nq}, {nk}, {d}
    x, w = torch.zeros(T, (nq + 2 * nk) * d, dtype=torch.bfloat16), torch.ones(d, dtype=torch.bfloat16)
    try:
        k.qk_norm_rope_bwd(x.clone(), x, w, w, torch.ones(T, nq + nk), None, T, nq, nk, d, torch.zeros(d), torch.zeros(d))
    except k.KernelError as e:
        print("refused", e)
"""


def _process(code, **sizes):
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code).format(**sizes)], capture_output=True, text=True)
    assert r.returncode == 0, f"the process ended with {r.returncode}: {r.stderr[-500:]}"
    return r.stdout


@pytest.mark.parametrize("d,nq,nk", [(528, 8, 2), (1024, 8, 2), (72, 8, 2), (0, 8, 2), (-16, 8, 2), (64, -1, 2), (64, 2, -1)])
def test_the_workspace_of_other_widths_is_refused_cpu(d, nq, nk):
    rc, floats, text = _process(WORKSPACE, T=256, nq=nq, nk=nk, d=d).split(maxsplit=2)
    assert int(rc) != 0 and int(floats) == -1 and "qk_norm_rope" in text


@pytest.mark.parametrize("d", [528, 1024, 72])
def test_the_backward_pass_of_other_widths_is_refused_cpu(d):
    assert "refused" in _process(BACKWARD, T=4, nq=2, nk=1, d=d)


def test_the_workspace_of_widths_it_takes_cpu():
    for d in (16, 64, 96, 512):
        floats = ctypes.c_long(0)
        assert k.lib().zb_qk_norm_rope_workspace(256, 8, 2, d, ctypes.addressof(floats)) == 0
        assert floats.value > 0 and floats.value % d == 0


@pytest.mark.parametrize("T,nq,nk,d", [(1, 2 ** 23, 0, 512), (1, 2 ** 22 - 192, 0, 512), (2, 2 ** 21, 2 ** 21, 512), (1, 2 ** 30, 2 ** 30, 16)])
def test_rows_beyond_32_bits_are_refused_cpu(T, nq, nk, d):
    """Before anything is launched, and before the library looks at an address."""
    L = k.lib()
    for rc in (L.zb_qk_norm_rope_fwd(0, 0, 0, 0, 0, 0, T, 1, nq, nk, nk, d, 2 ** 40, 2 ** 40, 1e-5, 0),
               L.zb_qk_norm_rope_bwd(0, 0, 0, 0, 0, 0, 0, 0, 0, T, 1, nq, nk, d, 2 ** 40, 2 ** 40, 1, 0)):
        assert rc == -1 and b" heads" in L.zb_last_error()


def test_heads_beyond_32_bits_are_refused_cpu(monkeypatch):
    """The wrapper: a number of heads that would reach the library as another one."""
    monkeypatch.setattr(k, "_bf16", lambda t, name: None)
    monkeypatch.setattr(k, "_on_current", lambda t, name: None)
    monkeypatch.setattr(k, "_lib", None)
    monkeypatch.setattr(k, "lib", lambda: pytest.fail("the library was reached"))
    w = torch.ones(16, dtype=torch.bfloat16)
    for nq, nk in ((2 ** 32 + 2, 0), (2 ** 31, 0), (-2, 2), (4, -1)):
        n = (nq + 2 * nk) * 16
        x = type("Rows", (), dict(shape=torch.Size((1, n)), dtype=torch.bfloat16, device=w.device, dim=lambda self: 2,
                                  stride=lambda self, i=None: (n, 1) if i is None else (n, 1)[i]))()
        with pytest.raises(ValueError, match="2\\^31"):
            k.qk_norm_rope_fwd(x, w, w, None, 1, nq, nk, 16, 1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [528, 1024, 72])
def test_both_passes_refuse_other_widths(d):
    from zorse_b200.ops.api import get_ops

    ops = get_ops("sm100")
    x, w = torch.zeros(4, 4 * d, dtype=torch.bfloat16, device="cuda"), torch.ones(d, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(k.KernelError):
        ops.qk_norm_rope_fwd(x, w, w, None, 4, 2, 1, d, 1e-5)
    with pytest.raises(k.KernelError):
        ops.qk_norm_rope_bwd(x.clone(), x, w, w, torch.ones(4, 3, device="cuda"), None, 4, 2, 1, d, torch.zeros(d, device="cuda"),
                             torch.zeros(d, device="cuda"))
