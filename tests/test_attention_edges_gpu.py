"""Attention at the edges that the shapes of test_attention_gpu.py leave out.  Its reference, tolerances and helpers hold here,
too, unless a test says otherwise."""
import pytest
import torch

from test_attention_gpu import compare, make

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
