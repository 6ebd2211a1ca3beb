"""The RMS norm's, SwiGLU's and the grouped products' entry points on the CPU host: malformed calls are refused with a
status and a message before any launch, and the operators refuse CPU tensors and wrong options."""

from __future__ import annotations

import pytest
import torch

P = 4096  # a 256-byte aligned stand-in address: every call below returns before using it


def test_module_has_the_operators():
    from lowbit import _lib

    mod = _lib.autograd()
    for fn in ("rms_norm", "rms_norm_quant", "swiglu", "grouped_matmul"):
        assert callable(getattr(mod, fn))
        with pytest.raises(TypeError, match="number of arguments"):
            getattr(mod, fn)(torch.ones(2, 4))


def test_operators_refuse_cpu_tensors():
    from lowbit.experts import grouped_matmul, local_moe_bf16, swiglu
    from lowbit.norm import RMSNorm, rms_norm, rms_norm_quant

    x, off = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    b = x.bfloat16()
    ids = torch.zeros(2, 1, dtype=torch.int32)
    for call in (lambda: rms_norm(x), lambda: rms_norm(x, residual=x), lambda: rms_norm_quant(x), lambda: RMSNorm(8)(x),
                 lambda: swiglu(x), lambda: grouped_matmul(b, b[None], off),
                 lambda: local_moe_bf16(b, ids, torch.ones(2, 1), torch.zeros(1, 256, 8).bfloat16(), torch.zeros(1, 8, 128).bfloat16())):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_expert_loop_runs_on_its_tensors_device(monkeypatch):
    """operands of two devices are refused, and every launch is made with theirs as the current one"""
    from lowbit import experts

    class Reached(Exception):
        pass

    current = []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            current.append(self.device)

        def __exit__(self, *exc):
            current.pop()

    def route(*a, **kw):
        raise Reached(list(current))

    monkeypatch.setattr(experts.ops, "_require_device", lambda *t: None)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(experts.moe, "route_by_expert", route)
    ok = [torch.zeros(2, 8).bfloat16(), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1),
          torch.zeros(1, 256, 8).bfloat16(), torch.zeros(1, 8, 128).bfloat16()]
    for i in range(5):
        with pytest.raises(ValueError, match="are on"):
            experts.local_moe_bf16(*(t.to("meta") if j == i else t for j, t in enumerate(ok)))
    with pytest.raises(Reached) as seen:
        experts.local_moe_bf16(*ok)
    assert seen.value.args[0] == [ok[0].device] and not current


def test_checkpoint_names():
    from lowbit import ops
    from lowbit.norm import RMSNorm

    assert ops.checkpoint_code(None) == 0 and ops.checkpoint_code("e4m3") == 1
    for bad in ("e5m2", "fp8", "", 1, True):
        with pytest.raises(ValueError, match="checkpoint"):
            RMSNorm(8, checkpoint=bad)


def test_rms_norm_validates_without_gpu():
    from lowbit import _lib

    L = _lib.lib()
    E, U = _lib.NTLB_EINVAL, _lib.NTLB_EUNSUPPORTED
    ok = dict(x=P, dt=0, T=4, H=64, ldx=64, res=None, ldr=64, w=P, wdt=0, eps=1e-6, s=None, lds=64, y=P, ldy=64, rstd=None,
              kept=None, ke=None)

    def fwd(**kw):
        a = {**ok, **kw}
        return L.ntlb_rms_norm_forward(*(a[k] for k in ok), None)

    for bad in (dict(x=None), dict(dt=7), dict(T=-1), dict(H=0), dict(ldx=63), dict(w=P, wdt=9), dict(eps=-1.0),
                dict(eps=float("nan")), dict(y=None), dict(ldy=63), dict(res=P), dict(s=P), dict(res=P, s=P, ldr=63),
                dict(res=P, s=P, lds=63), dict(kept=P), dict(ke=P), dict(kept=P + 8, ke=P)):
        assert fwd(**bad) == E and L.ntlb_last_error(), bad
    assert fwd(H=16385, ldx=16385, ldy=16385) == U

    okq = dict(x=P, dt=0, T=4, H=64, ldx=64, res=None, ldr=64, w=P, wdt=0, eps=1e-6, s=None, lds=64, grid=0, codes=P, ldc=128,
               scales=P, s_row=1, s_col=4, nan=None)

    def quant(**kw):
        a = {**okq, **kw}
        return L.ntlb_rms_norm_quant(*(a[k] for k in okq), None)

    for bad in (dict(x=None), dict(dt=7), dict(H=0), dict(ldx=63), dict(grid=9), dict(codes=None), dict(codes=P + 4),
                dict(ldc=64), dict(scales=None), dict(eps=-1.0), dict(res=P)):
        assert quant(**bad) == E and L.ntlb_last_error(), bad

    need = L.ntlb_rms_norm_workspace_bytes(0, 4, 64)
    assert need > 0 and L.ntlb_rms_norm_workspace_bytes(0, 0, 64) == 0
    okb = dict(s=P, dt=0, T=4, H=64, lds=64, kept=None, ke=None, dy=P, lddy=64, ds=None, ldds=64, rstd=P, w=P, wdt=0, dx=P,
               lddx=64, dw=P, ws=P, n=need)

    def bwd(**kw):
        a = {**okb, **kw}
        return L.ntlb_rms_norm_backward(*(a[k] for k in okb), None)

    for bad in (dict(dt=7), dict(H=0), dict(s=None), dict(s=None, kept=P), dict(lds=63), dict(dy=None), dict(lddy=63),
                dict(rstd=None), dict(dx=None), dict(lddx=63), dict(ds=P, ldds=63), dict(n=need - 1), dict(ws=None),
                dict(wdt=9)):
        assert bwd(**bad) == E and L.ntlb_last_error(), bad


def test_swiglu_validates_without_gpu():
    from lowbit import _lib

    L = _lib.lib()
    E = _lib.NTLB_EINVAL
    ok = dict(x=P, dt=0, T=4, I=256, ldx=512, block=0, h=P, ldh=256, kept=None, ke=None)

    def fwd(**kw):
        a = {**ok, **kw}
        return L.ntlb_swiglu_rows(*(a[k] for k in ok), None)

    for bad in (dict(x=None), dict(dt=7), dict(T=-1), dict(I=0), dict(ldx=511), dict(block=64), dict(block=-128),
                dict(block=384), dict(h=None), dict(ldh=255), dict(kept=P), dict(ke=P), dict(kept=P + 8, ke=P)):
        assert fwd(**bad) == E and L.ntlb_last_error(), bad
    okb = dict(x=P, dt=0, T=4, I=256, ldx=512, block=0, kept=None, ke=None, dh=P, lddh=256, dx=P, lddx=512)

    def bwd(**kw):
        a = {**okb, **kw}
        return L.ntlb_swiglu_rows_backward(*(a[k] for k in okb), None)

    for bad in (dict(x=None), dict(x=None, kept=P), dict(dt=7), dict(I=0), dict(ldx=511), dict(block=192), dict(dh=None),
                dict(lddh=255), dict(dx=None), dict(lddx=511)):
        assert bwd(**bad) == E and L.ntlb_last_error(), bad


def test_grouped_products_validate_without_gpu():
    from lowbit import _lib

    L = _lib.lib()
    E = _lib.NTLB_EINVAL
    sizes = dict(off=P, R=300, E=2, N=64, K=64)
    ok = {"y": dict(a=P, lda=64, w=P, ldw=64, ws=64 * 64, **sizes, out=P, ldo=64, buf=P, n=1 << 30),
          "dw": dict(a=P, lda=64, w=P, ldw=64, **sizes, out=P)}

    def call(which, **kw):
        a = {**ok["dw" if which == "dw" else "y"], **kw}
        fn = {"y": L.ntlb_grouped_matmul, "dx": L.ntlb_grouped_matmul_dx, "dw": L.ntlb_grouped_matmul_dw}[which]
        return fn(*a.values(), None)

    for which in ("y", "dx", "dw"):
        for bad in (dict(a=None), dict(a=P + 8), dict(lda=63), dict(lda=56), dict(lda=(1 << 22) + 8), dict(w=None), dict(ldw=60),
                    dict(off=None), dict(R=-1), dict(R=(1 << 30) + 1), dict(E=0), dict(E=4097), dict(N=0), dict(K=0),
                    dict(N=(1 << 22) + 1), dict(out=None)):
            assert call(which, **bad) in (E, _lib.NTLB_EUNSUPPORTED) and L.ntlb_last_error(), (which, bad)
        assert call(which, a=None) == E
    for which in ("y", "dx"):
        for bad in (dict(ws=4), dict(ws=-8), dict(ldo=63)):
            assert call(which, **bad) == E, (which, bad)
    # a contraction in ranges needs its sums' room: [ranges][R][N, a multiple of four]
    wide = dict(R=64, E=1, N=62, K=4096, lda=4096, ldw=4096)
    need = L.ntlb_grouped_matmul_workspace_bytes(64, 1, 62, 4096, 0)
    assert need > 0 and need % (64 * 64 * 4) == 0
    for bad in (dict(n=need - 1), dict(buf=None), dict(buf=P + 8)):
        assert call("y", **wide, **bad) == E and b"workspace" in L.ntlb_last_error(), bad
    need = L.ntlb_grouped_matmul_workspace_bytes(64, 1, 4096, 62, 1)
    assert need > 0
    assert call("dx", R=64, E=1, N=4096, K=62, lda=4096, n=need - 1) == E and b"workspace" in L.ntlb_last_error()
    assert L.ntlb_grouped_matmul_workspace_bytes(8, 1, 64, 4096, 0) == 0  # few rows: the weights stream past them
    assert L.ntlb_grouped_matmul_workspace_bytes(32768, 32, 4096, 7168, 0) == 0  # the tiles fill the chip
    assert L.ntlb_grouped_matmul_workspace_bytes(0, 1, 64, 64, 0) == L.ntlb_grouped_matmul_workspace_bytes(4, 0, 64, 64, 1) == 0


def test_grouped_products_of_too_many_tiles_are_refused():
    """a launch counts its threads in 32 bits: more tiles than that are refused before one"""
    from lowbit import _lib

    L = _lib.lib()
    U = _lib.NTLB_EUNSUPPORTED
    for R, E in ((5000, 4096), (1 << 30, 1)):
        wide = 1 << 22
        assert L.ntlb_grouped_matmul(P, 8, P, 8, 0, P, R, E, wide, 8, P, wide, None, 0, None) == U
        assert b"tiles" in L.ntlb_last_error()
        assert L.ntlb_grouped_matmul_dx(P, 8, P, wide, 0, P, R, E, 8, wide, P, wide, None, 0, None) == U
        assert b"tiles" in L.ntlb_last_error()


def test_kept_rows_validate_without_gpu():
    from lowbit import _lib

    L = _lib.lib()
    E = _lib.NTLB_EINVAL
    for a in ((P + 8, 64, 4, 64, P, P), (P, 60, 4, 64, P, P), (P, 64, -1, 64, P, P), (P, 64, 4, 0, P, P), (P, 64, 4, 64, None, P),
              (P, 64, 4, 64, P + 8, P), (P, 64, 4, 64, P, None)):
        assert L.ntlb_kept_rows(*a, None) == E and L.ntlb_last_error(), a
    for a in ((None, P, 4, 64, P, 64), (P, None, 4, 64, P, 64), (P, P, 4, 64, None, 64), (P, P, 4, 64, P, 60), (P, P, 4, 64, P, 56),
              (P, P, -1, 64, P, 64), (P, P, 4, 0, P, 64)):
        assert L.ntlb_kept_values(*a, None) == E and L.ntlb_last_error(), a
