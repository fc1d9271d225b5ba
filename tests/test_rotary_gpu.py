"""Rotary positions (ops.rotary, functional.rotary, ops.RotaryTable) against complex products in 64 bits.

Tolerances: half a step of the result's type, and before that fp32: a table entry, a product and a sum are each off by
2^-24, so at most 4 * 2^-24 * (|a| + |b|) for the pair (a, b)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def reference(x, pos, freq, interleaved, sign=1.0, amplitude=1.0):
    """(result in 64 bits, |a| + |b| of each element's pair)."""
    R = 2 * len(freq)
    y = x.double()
    pos = pos.expand(x.shape[0], -1) if pos.dim() == 1 else pos
    ang = pos.double().unsqueeze(-1) * freq.to(x.device)
    unit = torch.polar(torch.full_like(ang, amplitude), sign * ang).unsqueeze(2)
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
    z = torch.complex(a, b) * unit
    size = a.abs() + b.abs()
    join = (lambda p, q: torch.stack((p, q), -1).flatten(-2)) if interleaved else (lambda p, q: torch.cat((p, q), -1))
    return torch.cat((join(z.real, z.imag), y[..., R:]), -1), torch.cat((join(size, size), torch.zeros_like(y[..., R:])), -1)


def inside(got, ref, size, what):
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + torch.finfo(got.dtype).smallest_normal + 4 * U * size
    over = (got.double() - ref).abs() - tol
    assert got.shape == ref.shape and bool((over <= 0).all()), f"{what}: {over.max().item():.3g} over the tolerance"


def freqs(R, base=10000.0):
    return torch.tensor([base ** (-2 * i / R) for i in range(R // 2)], dtype=torch.float64)


CASES = [  # B, T, Hq, Hk, D, R
    (1, 1, 1, 1, 2, 2), (3, 1, 4, 2, 64, 64), (2, 33, 3, 1, 32, 16), (1, 7, 5, 5, 20, 10), (2, 17, 2, 2, 7, 6), (64, 1, 32, 8, 128, 128),
    (2, 130, 8, 2, 128, 64), (5, 9, 1, 3, 48, 34), (1, 300, 2, 1, 96, 32), (2, 1100, 4, 1, 16, 16)]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hk,D,R", CASES)
def test_rotation_and_its_inverse(B, T, Hq, Hk, D, R, interleaved, kind):
    from recommendsystem_amd import ops
    g = torch.Generator(device="cuda").manual_seed(B * 1000 + T * 10 + D)
    q = torch.randn(B, T, Hq, D, device="cuda", generator=g).to(TYPES[kind])
    k = torch.randn(B, T, Hk, D, device="cuda", generator=g).to(TYPES[kind])
    pos = torch.randint(0, 5000, (B, T), device="cuda", generator=g)
    table = ops.RotaryTable(5000, R, "cuda", interleaved=interleaved)
    for sign, p in ((1.0, pos), (-1.0, pos.int()), (1.0, pos[0])):
        oq, ok = ops.rotary(table, p, q, k, inverse=sign < 0)
        assert oq.is_contiguous() and ok.is_contiguous()
        inside(oq, *reference(q, p, freqs(R), interleaved, sign), "q")
        inside(ok, *reference(k, p, freqs(R), interleaved, sign), "k")
        assert torch.equal(ops.rotary(table, p, q, inverse=sign < 0), oq)
    table.check_positions()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_strided_inputs(kind):
    from recommendsystem_amd import ops
    qkv = torch.randn(3, 21, 12, 32, device="cuda").to(TYPES[kind])
    pos = torch.arange(40, device="cuda")[5:26]
    table = ops.RotaryTable(40, 32, "cuda")
    views = [qkv[:, :, :6], qkv[:, :, 6:8], qkv.transpose(1, 2)[:, :6].transpose(1, 2), qkv[:, :, ::3], qkv.flip(3),
             qkv.transpose(2, 3)[:, :, :12].transpose(2, 3)[..., :12], qkv.flatten(2)[:, :, 1:321].view(3, 21, 10, 32)]
    small = ops.RotaryTable(40, 12, "cuda")
    for v in views:
        t = table if v.shape[3] == 32 else small
        inside(ops.rotary(t, pos, v), *reference(v, pos, freqs(t.rotary_dim), False), str(v.stride()))
    every = torch.arange(42, device="cuda").view(21, 2)[:, 0]            # positions with a stride
    wide = ops.RotaryTable(42, 32, "cuda")
    inside(ops.rotary(wide, every, qkv), *reference(qkv, every, freqs(32), False), "strided positions")
    one = torch.full((1, 1), 7, device="cuda").expand(3, 21)
    inside(ops.rotary(wide, one, qkv), *reference(qkv, one, freqs(32), False), "one position for all")


def test_far_positions_keep_their_angles():
    """The angle of position 1 000 000 is taken in 64 bits (in 32 it would be off by up to 1/16)."""
    from recommendsystem_amd import ops
    table = ops.RotaryTable(1000001, 8, "cuda")
    pos = torch.tensor([999999, 1000000, 123457], device="cuda")
    q = torch.randn(1, 3, 2, 8, device="cuda")
    inside(ops.rotary(table, pos, q), *reference(q, pos, freqs(8), False), "q")


def test_scaled_tables():
    from recommendsystem_amd import ops
    q = torch.randn(2, 50, 3, 64, device="cuda")
    pos = torch.arange(400, 450, device="cuda")
    slow = ops.RotaryTable(512, 64, "cuda", factor=4.0)
    inside(ops.rotary(slow, pos, q), *reference(q, pos, freqs(64) / 4, False), "linear")
    parts = ops.RotaryTable(512, 64, "cuda", base=500.0, factor=8.0, original_positions=256, ramp=(1.0, 8.0), amplitude=1.25)
    want = []
    for f in freqs(64, 500.0).tolist():
        turns = 256 * f / (2 * math.pi)
        keep = 0.0 if turns <= 1 else 1.0 if turns >= 8 else (turns - 1) / 7
        want.append(f * (keep + (1 - keep) / 8))
    assert any(0 < (256 * f / (2 * math.pi) - 1) / 7 < 1 for f in freqs(64, 500.0).tolist())
    ref, size = reference(q, pos, torch.tensor(want, dtype=torch.float64), False, amplitude=1.25)
    # the frequencies of the two computations may differ in the last of 53 bits, times the position: nothing in fp32
    inside(ops.rotary(parts, pos, q), ref, size * 1.25, "by parts")


def test_gradients():
    """The backward is the inverse rotation of the incoming gradient, for q, k, or one of them; and against differences (the
    map is linear, so a difference is exact up to rounding)."""
    from recommendsystem_amd import functional as Fn
    from recommendsystem_amd import ops
    table = ops.RotaryTable(100, 12, "cuda", interleaved=True)
    pos = torch.randint(0, 100, (2, 9), device="cuda")
    q, k = (torch.randn(2, 9, h, 16, device="cuda", requires_grad=True) for h in (4, 2))
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    oq, ok = Fn.rotary(table, pos, q, k)
    dq, dk = torch.autograd.grad((oq * gq).sum() + (ok * gk).sum(), (q, k))
    inside(dq, *reference(gq, pos, freqs(12), True, -1.0), "dq")
    inside(dk, *reference(gk, pos, freqs(12), True, -1.0), "dk")
    oq, ok = Fn.rotary(table, pos, q, k)
    assert torch.equal(torch.autograd.grad((ok * gk).sum(), k)[0], dk)
    assert torch.equal(torch.autograd.grad((Fn.rotary(table, pos, q) * gq).sum(), q)[0], dq)
    v = torch.randn_like(q)
    diff = ((Fn.rotary(table, pos, q.detach() + v).double() - Fn.rotary(table, pos, q.detach() - v).double()) * gq).sum() / 2
    # 1152 terms of size about 1: the sums of roundings stay below 1152 * 16 * 2^-24
    assert abs(float(diff - (dq * v).double().sum())) <= 1152 * 16 * U


def test_positions_outside_the_table_are_found_and_read_row_zero():
    from recommendsystem_amd import ops
    table = ops.RotaryTable(10, 8, "cuda")
    q = torch.randn(1, 4, 2, 8, device="cuda")
    for dtype in (torch.int64, torch.int32):
        out = ops.rotary(table, torch.tensor([0, 10, -1, 9], device="cuda", dtype=dtype), q)
        assert torch.equal(out[:, 1:3], q[:, 1:3])
        with pytest.raises(IndexError):
            table.check_positions()
        table.check_positions()


def test_captured_and_replayed():
    from recommendsystem_amd import ops
    table = ops.RotaryTable(64, 32, "cuda")
    q, k = torch.randn(4, 10, 4, 32, device="cuda").bfloat16(), torch.randn(4, 10, 2, 32, device="cuda").bfloat16()
    pos = torch.zeros(4, 10, device="cuda", dtype=torch.int64)
    ops.rotary(table, pos, q, k)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        oq, ok = ops.rotary(table, pos, q, k)
    for i in range(3):
        pos.copy_(torch.randint(0, 64, (4, 10), device="cuda"))
        q.copy_(torch.randn(4, 10, 4, 32, device="cuda"))
        g.replay()
        wq, wk = ops.rotary(table, pos, q, k)
        torch.cuda.synchronize()
        assert torch.equal(oq, wq) and torch.equal(ok, wk)


def test_empty_and_refused():
    from recommendsystem_amd import ops
    from recommendsystem_amd._lib import RSError
    table = ops.RotaryTable(10, 8, "cuda")
    q = torch.randn(2, 3, 4, 8, device="cuda")
    pos = torch.arange(3, device="cuda")
    assert ops.rotary(table, pos[:0], q[:, :0]).shape == (2, 0, 4, 8)
    assert ops.rotary(table, pos, q, q[:, :, :0])[1].shape == (2, 3, 0, 8)
    bad = [lambda: ops.rotary(table, pos, q.double()), lambda: ops.rotary(table, pos, q[0]), lambda: ops.rotary(table, pos.float(), q),
           lambda: ops.rotary(table, pos[:2], q), lambda: ops.rotary(table, pos, q, q[:, :2]), lambda: ops.rotary(table, pos, q, q.half()),
           lambda: ops.rotary(table, pos, q[..., :6]), lambda: ops.rotary(table, pos.cpu(), q), lambda: ops.rotary(table, pos, q.cpu()),
           lambda: ops.rotary(ops.RotaryTable(10, 8, "cpu"), pos, q), lambda: ops.RotaryTable(10, 7, "cuda"),
           lambda: ops.RotaryTable(0, 8, "cuda"), lambda: ops.RotaryTable(10, 8, "cuda", factor=0.0),
           lambda: ops.RotaryTable(10, 8, "cuda", original_positions=5, ramp=(2.0, 2.0))]
    for f in bad:
        with pytest.raises(RSError):
            f()


def test_more_tokens_than_a_grid_dimension_holds():
    from recommendsystem_amd import ops
    T = (1 << 25) + 100                      # eight tokens to a workgroup: over 2^22 workgroups
    table = ops.RotaryTable(64, 2, "cuda")
    q = torch.randn(1, T, 1, 2, device="cuda").half()
    pos = (torch.arange(T, device="cuda") % 64).int()
    out = ops.rotary(table, pos, q)
    for part in (slice(0, 100), slice(T - 100, T)):
        inside(out[:, part], *reference(q[:, part], pos[part], freqs(2), False), "q")
