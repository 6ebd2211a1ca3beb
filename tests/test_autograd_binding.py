"""The C++ autograd module loads on the CPU host, takes its functions' addresses
from the loaded library only, and refuses malformed calls with Python errors."""

from __future__ import annotations

import ctypes

import pytest
import torch


def test_module_binds_to_the_loaded_library():
    from lowbit import _lib

    mod = _lib.autograd()
    assert mod is _lib.autograd()
    for fn in ("layer_norm", "route", "linear_xent"):
        assert callable(getattr(mod, fn))


def test_bind_refuses_an_incomplete_table():
    from lowbit import _lib

    mod = _lib.autograd()
    one = {"ntlb_last_error": ctypes.cast(_lib.lib().ntlb_last_error, ctypes.c_void_p).value}
    with pytest.raises(ValueError, match="no address of ntlb_layer_norm_forward"):
        mod.bind(one)
    with pytest.raises(TypeError):
        mod.bind([])
    _lib._autograd = None
    assert _lib.autograd() is mod  # bound again


def test_calls_refuse_wrong_arguments():
    from lowbit import _lib

    mod = _lib.autograd()
    with pytest.raises(TypeError, match="number of arguments"):
        mod.layer_norm(torch.ones(2, 3))
    with pytest.raises(TypeError, match="number of arguments"):
        mod.route(torch.ones(2, 3), None)
    with pytest.raises(TypeError, match="number of arguments"):
        mod.linear_xent()


def test_operators_refuse_cpu_tensors():
    from lowbit.loss import linear_cross_entropy
    from lowbit.norm import layer_norm
    from lowbit.router import route_tokens

    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="ROCm device"):
        layer_norm(x)
    with pytest.raises(RuntimeError, match="ROCm device"):
        route_tokens(x, 2)
    with pytest.raises(RuntimeError, match="ROCm device"):
        linear_cross_entropy(x.bfloat16(), x.bfloat16(), torch.zeros(2, dtype=torch.int64))


def test_entry_points_validate_without_gpu():
    """bad shapes, enums and workspaces: NTLB_EINVAL / NTLB_EUNSUPPORTED and a message, before any launch"""
    from lowbit import _lib

    L = _lib.lib()
    E, U = _lib.NTLB_EINVAL, _lib.NTLB_EUNSUPPORTED
    P = 4096  # a 256-byte aligned stand-in address: every call below returns before using it
    nf = L.ntlb_layer_norm_forward
    assert nf(P, 7, 4, 64, 64, P, P, 0, 1e-5, P, 64, None, None, None) == E
    assert nf(P, 0, 4, 0, 64, P, P, 0, 1e-5, P, 64, None, None, None) == E
    assert nf(P, 0, 4, 16385, 16385, P, P, 0, 1e-5, P, 16385, None, None, None) == U
    assert nf(P, 0, 4, 64, 63, P, P, 0, 1e-5, P, 64, None, None, None) == E and b"pitch" in L.ntlb_last_error()
    assert nf(P, 0, 4, 64, 64, P, P, 0, -1.0, P, 64, None, None, None) == E and b"eps" in L.ntlb_last_error()
    assert nf(P, 0, 4, 64, 64, P, P, 0, 1e-5, P, 64, P, None, None) == E
    nb = L.ntlb_layer_norm_backward
    need = L.ntlb_layer_norm_workspace_bytes(0, 4, 64)
    assert need > 0 and L.ntlb_layer_norm_workspace_bytes(0, 0, 64) == 0
    assert nb(P, 0, 4, 64, 64, P, 64, P, P, P, 0, P, 64, P, P, P, need - 1, None) == E
    assert b"workspace" in L.ntlb_last_error()
    rt = L.ntlb_route_topk
    ok = dict(dtype=0, T=4, E=32, ld=32, k=4, groups=1, kept=1)

    def route(**kw):
        a = {**ok, **kw}
        return rt(P, a["dtype"], a["T"], a["E"], a["ld"], a["k"], 0, None, a["groups"], a["kept"], 1, 1.0, P, P, None)

    for bad in (dict(dtype=9), dict(E=0), dict(E=1025, ld=1025), dict(k=0), dict(k=17), dict(k=33), dict(ld=31),
                dict(groups=5), dict(groups=32, kept=32), dict(groups=4, kept=5), dict(groups=8, kept=0),
                dict(groups=16, kept=1)):
        assert route(**bad) == E, bad
    xf = L.ntlb_linear_xent_forward
    need = L.ntlb_linear_xent_workspace_bytes(8, 64, 100, 0)
    assert xf(P, 64, P, 64, P, 1, 8, 64, 100, -100, 3, P, P, P, need, None) == E
    assert xf(P, 64, P + 8, 64, P, 1, 8, 64, 100, -100, 2, P, P, P, need, None) == E
    assert xf(P, 64, P, 60, P, 1, 8, 64, 100, -100, 2, P, P, P, need, None) == E
    assert xf(P, 64, P, 64, P, 1, 8, 64, 100, -100, 2, P, P, P, need - 1, None) == E
    assert b"workspace" in L.ntlb_last_error()
    assert xf(P, 64, P, 64, P, 1, 1 << 25, 64, 100, -100, 2, P, P, P, 1 << 40, None) == U
    xb = L.ntlb_linear_xent_backward
    need = L.ntlb_linear_xent_workspace_bytes(8, 64, 100, 1)
    assert xb(P, P, 64, 8, 64, 100, 2, P, P, 60, P, 64, P, need, None) == E
    assert xb(P, P, 64, 8, 64, 100, 2, P, P, 64, P, 64, P, need - 1, None) == E


def test_an_empty_batch_has_the_sizes_of_one_row():
    """the head loss's forward lays out one row of state where there is none, and its backward that row's workspace: the
    sizes named for an empty batch hold them"""
    from lowbit import _lib

    L = _lib.lib()
    for H in (1, 64, 72, 7168):
        assert L.ntlb_linear_xent_state_bytes(0, H) == L.ntlb_linear_xent_state_bytes(1, H) > 256
        for V in (1, 300, 131072):
            assert L.ntlb_linear_xent_workspace_bytes(0, H, V, 1) == L.ntlb_linear_xent_workspace_bytes(1, H, V, 1) > 0
            assert L.ntlb_linear_xent_workspace_bytes(0, H, V, 0) == 0
    assert L.ntlb_linear_xent_state_bytes(-1, 64) == L.ntlb_linear_xent_workspace_bytes(-1, 64, 64, 1) == 0
