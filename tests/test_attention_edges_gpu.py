"""Attention at the edges that the shapes of test_attention_gpu.py leave out.  Its reference, tolerances and helpers hold here,
too, unless a test says otherwise."""
import pytest
import torch

from test_attention_gpu import compare, inside, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Tk,D", [(64, 16), (48, 32), (32, 64), (16, 128)])
def test_turns_of_one_wave_do_not_meet_in_lds(kind, Tk, D):
    """Few keys, four row tiles for each of the four heads that share a key head: one wave takes them in turn through the same
    LDS tiles.  Right, and the same bits whatever else runs."""
    from recommendsystem_amd import ops
    q, k, v, do = make(70, 64, Tk, 8, 2, D, kind, seed=D)
    compare(q, k, v, do)
    compare(q, k, v, do, causal=True, query_start=Tk - 64)
    o, lse = ops.attention_fwd(q, k, v)
    first = (o, lse, *ops.attention_bwd(do, q, k, v, o, lse))
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                x = ops.attention_fwd(q, k, v)
                outs.append((*x, *ops.attention_bwd(do, q, k, v, *x)))
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, first))


@pytest.mark.parametrize("Tq,Tk,D", [(20, 30, 16), (70, 150, 24), (70, 40, 128)])
def test_rows_whose_scores_all_overflow_have_no_part_in_the_gradients(Tq, Tk, D):
    """fp32 products of -1e20 and 1e20 overflow to -inf.  Such rows get zeros and lse = -inf, as rows that see nothing; the other
    rows (q = 0: scores of zero) and the gradients of keys and values are as if they were not there."""
    from recommendsystem_amd import ops
    q, k, v, do = make(2, Tq, Tk, 2, 1, D, "f32", seed=41)
    k = 1e20 * (0.5 + torch.rand_like(k))
    lost = torch.arange(Tq, device="cuda") % 3 == 1
    q = torch.where(lost.view(1, -1, 1, 1), -1e20, 0.0).expand_as(q).contiguous()
    o, lse = ops.attention_fwd(q, k, v)
    got = (o, *ops.attention_bwd(do, q, k, v, o, lse))
    ref = reference(torch.zeros_like(q), k, v, torch.where(lost.view(1, -1, 1, 1), 0.0, do))
    assert torch.equal(lse == -torch.inf, lost.expand_as(lse))
    for name, x in zip(("o", "dq", "dk", "dv"), got):
        if name in ("o", "dq"):
            assert torch.count_nonzero(x[:, lost]).item() == 0, name
            inside(x[:, ~lost], ref[name][0][:, ~lost], ref[name][1][:, ~lost], name)
        else:
            inside(x, *ref[name], name)
