"""Layer norm at the edges that the shapes of test_layer_norm_gpu.py leave out.  Its reference and tolerances hold here, too,
unless a test says otherwise."""
import pytest
import torch

from test_layer_norm_gpu import U, compare, inside, make

pytestmark = pytest.mark.gpu


def test_more_parameter_sums_than_a_grid_dimension_holds():
    """Over 2^22 workgroups of 1024 lanes add the parameters' sums of a row of 2^26 elements: with one row, db is dy itself and
    dw is dy xhat of the kernel's own mean and rstd, three roundings."""
    from recommendsystem_amd import ops
    N = (1 << 26) + 33
    x = torch.randn(1, N, device="cuda").half()
    dy = torch.randn(1, N, device="cuda").half()
    _, s, mean, rstd = ops.layer_norm_fwd(x)
    _, dw, db = ops.layer_norm_bwd(dy, s, mean, rstd, param_dtype=torch.float32)
    assert torch.equal(db, dy[0].float())
    for part in (slice(0, 1000), slice(N // 2, N // 2 + 1000), slice(N - 1000, N)):
        ref = dy[0, part].double() * ((x[0, part].double() - mean.double()) * rstd.double())
        inside(dw[part], ref, 4 * U * ref.abs(), "dw")


@pytest.mark.parametrize("kind,wkind", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("M,N", [(2100, 5000), (1100, 16400), (2100, 4097), (1030, 16384), (3000, 1100)])
def test_workgroups_of_wide_rows_meet_several(M, N, kind, wkind):
    """More rows than the backward has workgroups: of one wide row each, and of a row longer than the registers hold."""
    compare(*make(M, N, kind, wkind, residual=N % 2 == 0, seed=M + N))


def test_wide_rows_at_odd_addresses():
    x, r, w, b, dy, ds = make(1500, 5003, "bf16", "f32", True, seed=77)
    compare(x[:, 2:], r[:, 1:-1], w[2:], b[2:].clone(), dy[:, :-2], ds[:, 2:])
