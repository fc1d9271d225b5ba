"""Layer norm with a residual stream (ops.layer_norm_fwd / _bwd, functional.layer_norm, layers.LayerNorm) against the
formulas in 64 bits.

Tolerances.  A result is rounded once to its type: half a step, finfo.eps / 2 relative.  Before that everything is fp32:
a sum runs over at most 16 terms in a lane and log2 of the lanes after that (under 32 additions), so mean and variance
are off by 32 roundings of the average magnitude, the normalised value by no more than 64 * 2^-24 * (1 + |xhat|), the
two row averages of the backward by as much of their own magnitudes.  dw and db add M rows in chains of under 256."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(t, ref):
    return torch.finfo(t).eps / 2 * ref.abs() + torch.finfo(t).smallest_normal


def inside(got, ref, tol, what):
    assert got.shape == ref.shape, what
    over = (got.double() - ref).abs() - tol
    assert bool((over <= 0).all()), f"{what}: {over.max().item():.3g} over the tolerance at {over.argmax().item()}"


def reference(x, r, w, b, dy, ds, eps):
    s = x if r is None else (x.double() + r.double()).to(x.dtype)
    z = s.double()
    N = z.shape[-1]
    c = z - z.mean(-1, keepdim=True)
    rs = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    xh = c * rs
    wd = torch.ones(N, device=x.device, dtype=torch.float64) if w is None else w.double()
    bd = torch.zeros(N, device=x.device, dtype=torch.float64) if b is None else b.double()
    out = {"s": s, "y": xh * wd + bd, "xh": xh, "wd": wd, "bd": bd, "rs": rs}
    if dy is not None:
        d = dy.double()
        g = d * wd
        dx = rs * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        out["dx"] = dx if ds is None else dx + ds.double()
        out["dx_scale"] = rs * (g.abs() + g.abs().mean(-1, keepdim=True) + (1 + xh.abs()) * (g * xh).abs().mean(-1, keepdim=True))
        flat = lambda t: t.reshape(-1, N)      # noqa: E731
        out["dw"], out["db"] = flat(d * xh).sum(0), flat(d).sum(0)
        out["dw_scale"], out["db_scale"] = flat(d.abs() * (1 + xh.abs())).sum(0), flat(d.abs()).sum(0)
    return out


def compare(x, r, w, b, dy, ds, eps=1e-5):
    from recommendsystem_amd import ops
    ref = reference(x, r, w, b, dy, ds, eps)
    y, s, mean, rstd = ops.layer_norm_fwd(x, w, b, eps, residual=r)
    assert torch.equal(s, ref["s"])
    inside(y, ref["y"], half_step(y.dtype, ref["y"]) + 64 * U * ((1 + ref["xh"].abs()) * ref["wd"].abs() + ref["bd"].abs()), "y")
    if dy is None:
        return
    dx, dw, db = ops.layer_norm_bwd(dy, s, mean, rstd, w, ds=ds, param_dtype=None if b is None else b.dtype)
    inside(dx, ref["dx"], half_step(dx.dtype, ref["dx"]) + 128 * U * ref["dx_scale"], "dx")
    inside(dw, ref["dw"], half_step(dw.dtype, ref["dw"]) + 256 * U * ref["dw_scale"], "dw")
    inside(db, ref["db"], half_step(db.dtype, ref["db"]) + 256 * U * ref["db_scale"], "db")


def make(M, N, kind, wkind, residual, seed=0, lead=()):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *sh, t=TYPES[kind]: torch.randn(*sh, device="cuda", generator=g).to(t)     # noqa: E731
    sh = (*lead, M, N)
    w, b = (1 + 0.3 * rn(N)).to(TYPES[wkind]), rn(N, t=TYPES[wkind])
    return 2 * rn(*sh) + 0.5, rn(*sh) if residual else None, w, b, rn(*sh), rn(*sh) if residual else None


# one row and many, widths around each lane count and vector, odd ones, beyond the register form
SHAPES = [(1, 1), (3, 2), (1, 16), (70, 39), (33, 64), (257, 128), (5, 129), (64, 513), (300, 777), (17, 1024), (9, 1030), (40, 4096),
          (3, 4104), (2, 16384), (3, 16385), (2, 20001)]


@pytest.mark.parametrize("kind,wkind", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("M,N", SHAPES)
def test_shapes_and_types(M, N, kind, wkind):
    compare(*make(M, N, kind, wkind, residual=(M + N) % 2 == 0, seed=M * 31 + N))


def test_many_rows_through_every_workgroup():
    compare(*make(5000, 48, "f32", "f32", True, seed=5))
    compare(*make(2500, 1000, "bf16", "f32", False, seed=6))
    compare(*make(1100, 2048, "f16", "f16", True, seed=7))


@pytest.mark.parametrize("have_w,have_b", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(have_w, have_b):
    x, r, w, b, dy, ds = make(37, 96, "bf16", "f32", True, seed=3)
    compare(x, r, w if have_w else None, b if have_b else None, dy, ds)


def test_leading_dimensions_strided_rows_and_unaligned_rows():
    x, r, w, b, dy, ds = make(7, 64, "f32", "f32", True, seed=4, lead=(3, 5))
    compare(x, r, w, b, dy, ds)
    wide = [t if t is None else torch.cat([t, t, t], -1) for t in (x, r, dy, ds)]
    for off in (64, 65, 1):                                  # a block of columns of wider rows, aligned and not
        xs, rr, dd, qq = (t[..., off:off + 64] for t in wide)
        assert not xs.is_contiguous()
        compare(xs, rr, w, b, dd, qq)
    compare(x.transpose(0, 1), r.transpose(0, 1), w, b, dy.transpose(0, 1), ds.transpose(0, 1))      # rows in no single stride
    compare(x.transpose(1, 3), None, w[:5].contiguous(), b[:5].contiguous(), dy.transpose(1, 3), None)      # elements apart
    compare(x[:1, :1, :1].expand(3, 5, 7, 64), r, w, b, dy[:1].expand(3, 5, 7, 64), ds)                  # one row for all


def test_large_mean_and_constant_rows():
    """The variance is that of centred values: a mean 1000 times the spread costs the input's own rounding and no more."""
    from recommendsystem_amd import ops
    g = torch.Generator(device="cuda").manual_seed(8)
    x = 1000 + torch.randn(33, 512, device="cuda", generator=g)
    y = ops.layer_norm_fwd(x)[0]
    ref = reference(x, None, None, None, None, None, 1e-5)["y"]
    # the mean (about 1000) is off by at most 32 roundings of its size, the rest as in the header
    inside(y, ref, half_step(torch.float32, ref) + 64 * U * (1 + ref.abs()) + 32 * U * 1000, "y")
    c = torch.full((4, 300), 3.0, device="cuda")
    y, _, mean, rstd = ops.layer_norm_fwd(c)
    # 300 equal values: their sum is exact, so is the mean, up to the one division
    assert bool((y.abs() <= 3 * U / 1e-5 ** 0.5).all()) and bool(torch.isfinite(rstd).all())


def test_no_rows():
    from recommendsystem_amd import ops
    x = torch.empty(0, 40, device="cuda")
    y, s, mean, rstd = ops.layer_norm_fwd(x)
    assert y.shape == (0, 40) and mean.numel() == 0
    dx, dw, db = ops.layer_norm_bwd(x, x, mean, rstd)
    assert dx.shape == (0, 40) and torch.count_nonzero(dw).item() == 0 and torch.count_nonzero(db).item() == 0


def test_a_nan_stays_in_its_row():
    from recommendsystem_amd import ops
    x = torch.randn(70, 130, device="cuda")
    clean = ops.layer_norm_fwd(x)[0]
    x[13, 7] = float("nan")
    y = ops.layer_norm_fwd(x)[0]
    rows = torch.arange(70, device="cuda") != 13
    assert torch.equal(y[rows], clean[rows]) and bool(torch.isnan(y[13]).all())


def test_module_and_autograd():
    """layers.LayerNorm: nn.LayerNorm's state_dict, and its gradients with a residual used twice; parameters that do not
    require gradients get none; a result nobody uses costs nothing."""
    from recommendsystem_amd.layers import LayerNorm
    torch.manual_seed(9)
    m = LayerNorm(48).cuda()
    ref = torch.nn.LayerNorm(48).cuda().double()
    with torch.no_grad():
        m.weight.uniform_(0.5, 1.5)
        m.bias.normal_()
    ref.load_state_dict({k: v.double() for k, v in m.state_dict().items()})
    x = torch.randn(4, 19, 48, device="cuda", requires_grad=True)
    r = torch.randn(4, 19, 48, device="cuda", requires_grad=True)
    gy, gs = torch.randn(4, 19, 48, device="cuda"), torch.randn(4, 19, 48, device="cuda")
    y, s = m(x, r)
    got = torch.autograd.grad((y * gy + s * gs).sum(), (x, r, m.weight, m.bias))
    xd, rd = x.detach().double().requires_grad_(), r.detach().double().requires_grad_()
    sd = xd + rd
    want = torch.autograd.grad((ref(sd) * gy + sd * gs).sum(), (xd, rd, ref.weight, ref.bias))
    for a, b in zip(got, want):
        # sums of up to 76 terms of size below 20 each, 300 roundings of fp32 at most
        torch.testing.assert_close(a.double(), b, rtol=300 * U, atol=300 * U * 20)
    y, s = m(x, r)
    only = torch.autograd.grad((s * gs).sum(), (x, r, m.weight), allow_unused=True)
    assert torch.equal(only[0], gs) and torch.equal(only[1], gs) and torch.count_nonzero(only[2]).item() == 0
    m.requires_grad_(False)
    assert torch.equal(torch.autograd.grad((m(x) * gy).sum(), x)[0].isfinite().all(), torch.tensor(True, device="cuda"))


def test_gradient_against_differences():
    from recommendsystem_amd import functional as Fn
    torch.manual_seed(10)
    x = torch.randn(3, 24, device="cuda", requires_grad=True)
    w = (1 + 0.2 * torch.randn(24, device="cuda")).requires_grad_()
    b = torch.randn(24, device="cuda", requires_grad=True)
    gy = torch.randn(3, 24, device="cuda")
    f = lambda *a: (Fn.layer_norm(*a) * gy).double().sum()      # noqa: E731
    grads = torch.autograd.grad(f(x, w, b), (x, w, b))
    h = 2.0 ** -8
    for i, t in enumerate((x, w, b)):
        v = torch.randn_like(t)
        v /= v.norm()
        args = [a.detach().clone() for a in (x, w, b)]
        args[i] = t.detach() + h * v
        up = f(*args)
        args[i] = t.detach() - h * v
        diff = (up - f(*args)) / (2 * h)
        # 72 products of about 1, each off by 64 roundings, over 2h; the third derivative over h^2 / 6 is below h
        assert abs(float(diff - (grads[i] * v).double().sum())) <= 72 ** 0.5 * 8 * 64 * U / h + 4 * h * h * 72 ** 0.5


def test_same_bits_every_time_on_two_streams_and_in_a_replayed_graph():
    from recommendsystem_amd import ops
    x, r, w, b, dy, ds = make(3000, 200, "bf16", "f32", True, seed=11)

    def step():
        y, s, mean, rstd = ops.layer_norm_fwd(x, w, b, residual=r)
        return y, s, *ops.layer_norm_bwd(dy, s, mean, rstd, w, ds=ds)

    first = [t.clone() for t in step()]
    a, c = torch.cuda.Stream(), torch.cuda.Stream()
    for st in (a, c):
        st.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(4):
        for st in (a, c):
            with torch.cuda.stream(st):
                outs.append(step())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, first))
    graphs = []
    for _ in range(2):                                       # two graphs over the same inputs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for seed in (1, 2, 3):
        x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        for g, _ in graphs:
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_refusals():
    from recommendsystem_amd import ops
    from recommendsystem_amd._lib import RSError
    from recommendsystem_amd.layers import LayerNorm
    x = torch.randn(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    bad = [lambda: ops.layer_norm_fwd(x.double()), lambda: ops.layer_norm_fwd(x.long()), lambda: ops.layer_norm_fwd(x, w[:7]),
           lambda: ops.layer_norm_fwd(x, w.bfloat16()), lambda: ops.layer_norm_fwd(x.bfloat16(), w, w.bfloat16()),
           lambda: ops.layer_norm_fwd(x, residual=x[:3]), lambda: ops.layer_norm_fwd(x, residual=x.half()),
           lambda: ops.layer_norm_fwd(x, w.cpu()), lambda: ops.layer_norm_fwd(x.cpu()), lambda: ops.layer_norm_fwd(x[:, :0]),
           lambda: ops.layer_norm_fwd(x, torch.ones(16, device="cuda")[::2]),
           lambda: ops.layer_norm_bwd(x, x, w[:4], w[:3], w), lambda: ops.layer_norm_bwd(x[:, :4], x, w[:4], w[:4], w),
           lambda: LayerNorm(9).cuda()(x), lambda: LayerNorm((4, 8))]
    for f in bad:
        with pytest.raises(RSError):
            f()


def test_more_rows_than_a_grid_dimension_holds():
    from recommendsystem_amd import ops
    M = (1 << 27) + 1000                     # 32 rows to a workgroup: over 2^22 workgroups
    x = torch.randn(M, 2, device="cuda").half()
    b = torch.tensor([0.5, -2.0], device="cuda").half()
    y, _, mean, rstd = ops.layer_norm_fwd(x, None, b)
    for part in (slice(0, 100), slice(M - 100, M)):
        ref = reference(x[part], None, None, b, None, None, 1e-5)
        inside(y[part], ref["y"], half_step(y.dtype, ref["y"]) + 64 * U * (1 + ref["xh"].abs() + ref["bd"].abs()), "y")
