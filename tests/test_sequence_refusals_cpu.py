"""Refusals of the sequence operators' entry points that need no GPU: every argument error is found on the host, before a
launch, and CPU tensors are rejected."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(256)             # never dereferenced: the calls are refused on their other arguments


def lib():
    from recommendsystem_amd import _lib
    return _lib.lib()


def refused(rc, code, word):
    assert rc == code and word in lib().rs_last_error_string(), (rc, lib().rs_last_error_string())


def ln_fwd(dtype=0, pdt=0, x=P, ldx=8, r=None, ldr=0, M=4, N=8, y=P, s=None):
    return lib().rs_layer_norm_fwd(dtype, pdt, x, ldx, r, ldr, M, N, None, None, 1e-5, y, s, None, None, None)


def ln_bwd(dtype=0, pdt=0, dy=P, s=P, lds=8, ds=None, ldds=0, M=4, N=8, dx=P, dw=None, work=None, floats=0):
    return lib().rs_layer_norm_bwd(dtype, pdt, dy, 8, s, lds, P, P, None, ds, ldds, M, N, dx, dw, None, work, floats, None)


def rotary(dtype=0, q=P, Hq=2, k=None, Hk=0, B=1, T=2, D=8, R=8, pos=P, cos=P, maxp=16, qo=P, ko=None):
    return lib().rs_rotary(dtype, q, 32, 16, 8, Hq, k, 32, 16, 8, Hk, B, T, D, R, 0, pos, 1, 0, 1, cos, P, maxp, 0, qo, ko, P, None)


def att_fwd(dtype=0, q=P, k=P, B=1, Tq=2, Tk=3, Hq=2, Hk=1, D=8, scale=1.0, o=P, work=None, floats=0):
    return lib().rs_attention_fwd(dtype, q, 0, 16, 8, k, 0, 8, 8, P, 0, 8, 8, B, Tq, Tk, Hq, Hk, D, None, None, 0, None, 0, scale, o, None,
                                  work, floats, None)


def att_bwd(dtype=0, go=P, B=1, Tq=2, Tk=3, Hq=2, Hk=1, D=8, scale=1.0, dq=P, work=None, floats=0):
    s = (0, 16, 8)
    return lib().rs_attention_bwd(dtype, go, *s, P, *s, P, *s, P, *s, P, *s, P, B, Tq, Tk, Hq, Hk, D, None, None, 0, None, 0, scale, dq, P, P,
                                  work, floats, None)


def test_layer_norm_refusals():
    refused(ln_fwd(dtype=3), -1, b"type")
    refused(ln_fwd(dtype=0, pdt=1), -1, b"type")
    refused(ln_fwd(dtype=1, pdt=2), -1, b"type")
    refused(ln_fwd(N=0), -1, b"shape")
    refused(ln_fwd(M=-1), -1, b"shape")
    refused(ln_fwd(x=None), -1, b"null")
    refused(ln_fwd(r=P, ldr=8, s=None), -1, b"null")
    refused(ln_fwd(ldx=7), -1, b"stride")
    refused(ln_fwd(r=P, ldr=3, s=P), -1, b"stride")
    assert ln_fwd(M=0, x=None, y=None) == 0
    refused(ln_bwd(dtype=5), -1, b"type")
    refused(ln_bwd(dx=None), -1, b"null")
    refused(ln_bwd(lds=4), -1, b"stride")
    refused(ln_bwd(ds=P, ldds=7), -1, b"stride")
    refused(ln_bwd(dw=P), -3, b"workspace")
    need = lib().rs_layer_norm_bwd_workspace_floats(4, 8)
    assert need >= 16
    refused(ln_bwd(dw=P, work=P, floats=need - 1), -3, b"workspace")


def test_rotary_refusals():
    refused(rotary(dtype=-1), -1, b"type")
    refused(rotary(R=7), -1, b"shape")
    refused(rotary(R=0), -1, b"shape")
    refused(rotary(R=10), -1, b"shape")
    refused(rotary(maxp=0), -1, b"shape")
    refused(rotary(q=None), -1, b"null")
    refused(rotary(k=P, Hk=1), -1, b"null")
    refused(rotary(pos=None), -1, b"null")
    refused(rotary(cos=None), -1, b"null")
    refused(rotary(Hq=1 << 24), -1, b"too many")
    refused(rotary(B=1 << 20, T=1 << 20), -1, b"too many")
    assert rotary(T=0, q=None, qo=None) == 0 and rotary(Hq=0, q=None, qo=None) == 0


def test_attention_refusals():
    for f in (att_fwd, att_bwd):
        refused(f(dtype=3), -1, b"type")
        refused(f(D=129), -1, b"shape")
        refused(f(D=0), -1, b"shape")
        refused(f(Hq=3, Hk=2), -1, b"shape")
        refused(f(Hk=0), -1, b"shape")
        refused(f(Tq=-1), -1, b"shape")
        refused(f(scale=0.0), -1, b"scale")
        refused(f(scale=float("nan")), -1, b"scale")
        refused(f(scale=float("inf")), -1, b"scale")
        refused(f(Tk=(1 << 30) + 1), -1, b"too large")
        refused(f(B=1 << 30, Hq=64, Hk=64), -1, b"too large")
        assert f(B=0) == 0
    refused(att_fwd(q=None), -1, b"null")
    refused(att_fwd(k=None), -1, b"null")
    refused(att_bwd(go=None), -1, b"null")
    refused(att_bwd(dq=None), -1, b"null")
    need = lib().rs_attention_fwd_workspace_floats(0, 1, 1, 100000, 2, 1, 8)
    assert need > 0 and lib().rs_attention_fwd_workspace_floats(0, 1, 1, 30, 2, 1, 8) == 0
    refused(att_fwd(Tq=1, Tk=100000), -3, b"workspace")
    refused(att_fwd(Tq=1, Tk=100000, work=P, floats=need - 1), -3, b"workspace")
    refused(att_fwd(Tq=1, Tk=100000, work=ctypes.c_void_p(260), floats=need), -1, b"aligned")
    refused(att_bwd(Tq=500, Tk=500), -3, b"workspace")


def test_cpu_tensors_and_bad_arguments_are_rejected():
    from recommendsystem_amd import functional as Fn
    from recommendsystem_amd import interactions as X
    from recommendsystem_amd import ops
    from recommendsystem_amd._lib import RSError
    from recommendsystem_amd.layers import LayerNorm
    x, q = torch.zeros(3, 8), torch.zeros(1, 2, 2, 8)
    table = ops.RotaryTable(4, 8, "cpu")
    pos = torch.arange(2)
    for f in (lambda: ops.layer_norm_fwd(x), lambda: Fn.layer_norm(x), lambda: LayerNorm(8)(x), lambda: ops.layer_norm_bwd(x, x, x[:, 0], x[:, 0]),
              lambda: ops.rotary(table, pos, q), lambda: Fn.rotary(table, pos, q), lambda: ops.attention_fwd(q, q, q),
              lambda: X.attention(q, q, q), lambda: ops.layer_norm_fwd(x.long()), lambda: ops.attention_fwd(q, q, q[:, :1]),
              lambda: ops.RotaryTable(4, 3, "cpu"), lambda: LayerNorm((2, 8))):
        with pytest.raises(RSError):
            f()


def test_rotary_table_values():
    from recommendsystem_amd import ops
    t = ops.RotaryTable(100, 6, "cpu", base=100.0)
    for p in (0, 1, 99):
        for i in range(3):
            a = p * 100.0 ** (-2 * i / 6)
            c, s = torch.tensor(a, dtype=torch.float64).cos(), torch.tensor(a, dtype=torch.float64).sin()
            # one rounding to fp32; the angle's own is of 53 bits
            assert abs(float(t.cos[p, i]) - float(c)) <= 2.0 ** -24 and abs(float(t.sin[p, i]) - float(s)) <= 2.0 ** -24
