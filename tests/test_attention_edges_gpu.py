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


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Tq,Tk,D", [(20, 30, 16), (70, 150, 64), (130, 40, 128), (3, 4000, 64)])
def test_rows_that_see_nothing_stay_zero_beside_rows_of_infinite_keys(Tq, Tk, D, kind):
    """A non-finite key or value is the business of the rows that see it: rows behind the sample's own and rows in front of
    its first key get zeros even where they share a tile with such rows."""
    from recommendsystem_amd import ops
    q, k, v, do = make(2, Tq, Tk, 4, 2, D, kind, seed=51)
    n = torch.tensor([Tq - 1, Tq - 2], device="cuda", dtype=torch.int32)
    i = torch.arange(Tq, device="cuda").view(1, -1)
    for name, t in (("v", v), ("k", k)):
        for fill in (float("inf"), float("nan")):
            x = t.clone()
            x[:, 0] = fill
            kv = (k, x) if name == "v" else (x, v)
            for how, out in ((dict(query_lengths=n), i >= n.view(-1, 1)), (dict(causal=True, query_start=-1), (i < 1).expand(2, -1))):
                o, lse = ops.attention_fwd(q, *kv, **how)
                dq = ops.attention_bwd(do, q, *kv, o, lse, **how)[0]
                assert torch.equal(lse == -torch.inf, out.view(2, 1, Tq).expand_as(lse))
                assert torch.count_nonzero(o[out]).item() == 0 and torch.count_nonzero(dq[out]).item() == 0, (name, fill, how)
