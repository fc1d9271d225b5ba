"""Attention at the edges that the shapes of test_attention_gpu.py leave out.  Its reference, tolerances and helpers hold here,
too, unless a test says otherwise."""
import pytest
import torch

from test_attention_gpu import U, compare, half_step, inside, make, reference

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


# fp16 gradients.  dS is rounded once and averages over the terms it is summed with like the result's own rounding, P as well
# (dv), and so does o's in delta: sqrt(1 + 1 + 0.6) = 1.6 times the root mean square of one final rounding, whatever the size
# of the gradients.  Held to twice that rounding.  (With dS and P as they are, fp16 loses their last bits below 2^-14.)
def rounding(ref):
    return (ref.half().double() - ref).square().sum(-1).sqrt()


def off(got, ref):
    return (got.double() - ref).square().sum(-1).sqrt()


def gradients(q, k, v, do, **how):
    from recommendsystem_amd import ops
    o, lse = ops.attention_fwd(q, k, v, **how)
    ref = reference(q, k, v, do, **how)
    return [(n, g, ref[n][0]) for n, g in zip(("dq", "dk", "dv"), ops.attention_bwd(do, q, k, v, o, lse, **how))]


@pytest.mark.parametrize("size", [1e-1, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("B,T,Hq,Hk,D", [(1, 2048, 2, 1, 128), (1, 2048, 2, 1, 64), (3, 200, 4, 4, 32), (5, 60, 2, 1, 64), (6, 31, 2, 2, 128)])
def test_fp16_gradients_of_any_size(B, T, Hq, Hk, D, size):
    q, k, v, do = make(B, T, T, Hq, Hk, D, "f16", seed=T + D)
    for name, got, ref in gradients(q, k, v, (do * size).half()):
        assert off(got, ref).square().sum() <= 4 * rounding(ref).square().sum(), name


@pytest.mark.parametrize("B,T,D", [(1, 700, 128), (1, 700, 64), (4, 60, 64)])
def test_fp16_gradients_of_every_row_where_rows_differ(B, T, D):
    """Rows whose gradients lie a factor of 10^4 apart: each row of dq by itself (64 or 128 elements of a row: up to three times
    its rounding), dk and dv as a whole."""
    q, k, v, do = make(B, T, T, 2, 1, D, "f16", seed=61)
    do = (do * 10.0 ** -(torch.arange(T, device="cuda") * 7 % 5).view(1, -1, 1, 1)).half()
    for name, got, ref in gradients(q, k, v, do):
        if name == "dq":
            assert bool((off(got, ref) <= 3 * rounding(ref)).all()), (off(got, ref) / rounding(ref)).max()
        assert off(got, ref).square().sum() <= 4 * rounding(ref).square().sum(), name


@pytest.mark.parametrize("B,T,D", [(2, 300, 128), (2, 300, 64), (3, 60, 64), (3, 30, 128)])
def test_fp16_gradients_whose_terms_pass_the_type(B, T, D):
    """dS beyond 65504 whose sums with small keys and queries are ordinary numbers."""
    q, k, v, do = make(B, T, T, 2, 1, D, "f16", seed=62)
    q, k, v, do = (q / 1024).half(), (k / 1024).half(), (v * 4096).half(), (do * 4096).half()
    ds = (do.double().amax() * v.double().amax() / T * D ** 0.5)
    assert ds > 65504
    for name, got, ref in gradients(q, k, v, do):
        assert bool(ref.abs().amax() < 65504)
        assert off(got, ref).square().sum() <= 4 * rounding(ref).square().sum(), name


@pytest.mark.parametrize("Tq,Tk,D", [(40, 3000, 64), (1, 5000, 128), (40, 60, 64), (130, 2000, 32)])
def test_fp16_small_probabilities_keep_their_bits(Tq, Tk, D):
    """One key takes nearly all and holds nothing, the others have 2^-20 each and all the value: o is their sum, off by a half
    step for theirs and one for its own."""
    from recommendsystem_amd import ops
    q, k = (torch.zeros(2, t, 1, D, device="cuda").half() for t in (Tq, Tk))
    q[..., 0] = 1
    k[:, 7, 0, 0] = 14.2
    v = torch.zeros(2, Tk, 1, D, device="cuda").half()
    v[:] = (1000 * torch.rand(1, 1, 1, D, device="cuda") + 100).half()
    v[:, 7] = 0
    do = torch.full_like(q, 1024.0)
    o, lse = ops.attention_fwd(q, k, v, scale=1.0)
    ref = reference(q, k, v, do, scale=1.0)
    inside(o, ref["o"][0], 2.1 * half_step(torch.float16, ref["o"][0]), "o")
    inside(lse, *ref["lse"], "lse")
    dv = ops.attention_bwd(do, q, k, v, o, lse, scale=1.0)[2]
    # dv: the same two half steps; beyond 65520 (the one key's, over 1024 x 64 rows) the type's value is infinite
    past = ref["dv"][0].abs() >= 65520
    assert bool((dv[past] == torch.inf).all()) and bool(past.any()) == (Tq > 64)
    inside(dv[~past], ref["dv"][0][~past], 2.1 * half_step(torch.float16, ref["dv"][0][~past]), "dv")


def backward_floats(kind, q, k):
    """The large kernels' backward keeps delta in a workspace, the ones for few keys need none."""
    from recommendsystem_amd import _lib
    (B, Tq, Hq, D), (Tk, Hk) = q.shape, k.shape[1:3]
    return _lib.lib().rs_attention_bwd_workspace_floats(("f32", "bf16", "f16").index(kind), B, Tq, Tk, Hq, Hk, D, 0)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,D", [(150, 64), (150, 128), (45, 32)])
def test_strides_and_orders_of_both_sizes(T, D, kind):
    """The strides of a user's tensors, for the kernels that take tiles through buffer descriptors and those for few keys."""
    B, H = 2, 6
    g = torch.Generator(device="cuda").manual_seed(T + D)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(make(1, 1, 1, 1, 1, 1, kind, 0)[0].dtype)      # noqa: E731
    qkv, do = rn(B, T, 3 * H, D), rn(B, T, H, D)
    assert (backward_floats(kind, qkv[:, :, :H], qkv[:, :, H:2 * H]) > 0) == (T > 64)
    compare(qkv[:, :, :H], qkv[:, :, H:2 * H], qkv[:, :, 2 * H:], do)
    heads_first = qkv.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    compare(heads_first[:, :, :H], heads_first[:, :, H:H + 2], heads_first[:, :, -2:], do.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3))
    n = D - 5
    compare(qkv[..., 1:n + 1][:, :, :H], qkv[..., 2:n + 2][:, :, H:2 * H], qkv[..., 3:n + 3][:, :, 2 * H:], do[..., :n], causal=True)      # unaligned
    n = D - 8
    compare(qkv[..., 1:n + 1][:, :, :H], qkv[..., 2:n + 2][:, :, H:2 * H], qkv[..., 3:n + 3][:, :, 2 * H:], do[..., :n], causal=True)
    dims = qkv.transpose(2, 3)                                                            # last dimension not contiguous
    compare(dims[..., :8][:, :, :4], dims[..., 8:16][:, :, :2], dims[..., 2:10][:, :, :2], do.transpose(2, 3)[:, :, :4, :6].repeat(1, 1, 1, 2)[..., :8])
    compare(qkv[:1, :, :H].expand(B, T, H, D), qkv[:, :1, :H].expand(B, T, H, D), qkv[:, :, :1].expand(B, T, H, D), do[:, :1].expand(B, T, H, D))
    compare(qkv[:, :, :H], qkv[:1, :, :1].expand(B, T, H, D), qkv[:1, :, 1:2].expand(B, T, H, D), do[:, :, :1].expand(B, T, H, D))
    compare(qkv.flip(1)[:, :, :H], qkv[:, ::3, H:2 * H], qkv[:, 1:T:3, 2 * H:][:, :T // 3 + T % 3], do)
    wide = rn(B, T, 3 * H, 2 * D)                                                         # every second head, half of each, from a column on
    compare(wide[:, :, 0:2 * H:2, :D], wide[:, :, 1:2 * H:2, D:], wide[:, :, 2 * H:, D // 2:D // 2 + D], do)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("Tq,D", [(1, 64), (3, 128), (40, 64)])
def test_strides_of_a_cache(Tq, D, kind):
    """Few rows over a long cache that lies inside a wider one, heads first, with an expanded key head, unaligned."""
    B, Tk, H = 2, 3000, 2
    q, k, v, _ = make(B, Tq, Tk, 2 * H, H, D, kind, seed=71)
    wide = torch.randn(B, Tk + 100, 2 * H, D + 3, device="cuda").to(q.dtype)
    compare(q, wide[:, 50:50 + Tk, :H, :D], wide[:, 50:50 + Tk, H:, 3:], None)
    hf = lambda x: x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)                 # noqa: E731
    compare(hf(q), hf(k), hf(v), None, causal=True)
    compare(q, k[:, :, :1].expand(B, Tk, H, D), v[:1].expand(B, Tk, H, D), None)
    compare(q[..., 1:D - 2], k[..., 1:D - 2], v[..., 3:], None)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("Tq,D", [(150, 64), (150, 128), (1, 64), (40, 64)])
def test_far_offsets(Tq, D, kind):
    """Samples 2^31 elements apart, and rows 2^22 and more apart (past what a descriptor's tile may span): keys of a cache whose
    rows hold every layer."""
    T, B, H = 150, 2, 2
    far = (1 << 31) + 4096
    dtype = make(1, 1, 1, 1, 1, 1, kind, 0)[0].dtype
    store = torch.empty(far + T * 3 * H * D, device="cuda", dtype=dtype)
    qkv = store.as_strided((B, T, 3 * H, D), (far, 3 * H * D, D, 1))
    qkv.copy_(torch.randn(B, T, 3 * H, D, device="cuda"))
    do = torch.randn(B, Tq, H, D, device="cuda").to(dtype)
    assert backward_floats(kind, do, qkv[:, :, H:2 * H]) > 0
    compare(qkv[:, :Tq, :H], qkv[:, :, H:2 * H], qkv[:, :, 2 * H:], do, causal=True)
    del store, qkv
    for apart in ((1 << 22) - 8, 1 << 22, (1 << 24) + 8):        # the widest rows of the asynchronous loads, and past them
        store = torch.empty((T + 1) * apart, device="cuda", dtype=dtype)
        rows = store.as_strided((1, T, 3 * H, D), (T * apart, apart, D, 1))
        rows.copy_(torch.randn(1, T, 3 * H, D, device="cuda"))
        compare(rows[:, :Tq, :H], rows[:, :, H:2 * H], rows[:, :, 2 * H:], do[:1])
        del store, rows


@pytest.mark.parametrize("kind,D", [("bf16", 100), ("f16", 100), ("f32", 127), ("bf16", 65), ("f32", 102), ("f16", 127)])
@pytest.mark.parametrize("Tq,Tk", [(150, 150), (50, 150), (50, 50), (130, 64)])
def test_backward_of_wide_heads_that_are_not_aligned(Tq, Tk, D, kind):
    q, k, v, do = make(2, Tq, Tk, 4, 2, D, kind, seed=D + Tq)
    compare(q, k, v, do)
    compare(q, k, v, do, causal=True)
    n = torch.tensor([Tk, Tk // 3], device="cuda", dtype=torch.int32)
    compare(q, k, v, do, lengths=n, query_lengths=n.clamp(max=Tq), causal=True)


@pytest.mark.parametrize("Tq,G,D", [(1, 4, 7), (1, 1, 63), (2, 8, 7), (5, 3, 63), (1, 2, 33), (3, 1, 101), (1, 16, 30)])
def test_single_tokens_of_odd_heads_in_fp32(Tq, G, D):
    B, Tk, Hk = 3, 1003, 2
    q, k, v, _ = make(B, Tq, Tk, G * Hk, Hk, D, "f32", seed=D)
    n = torch.tensor([1003, 0, 517], device="cuda", dtype=torch.int32)
    compare(q, k, v, None)
    compare(q, k, v, None, lengths=n)
    compare(q, k, v, None, causal=True)
    pad = lambda x: torch.nn.functional.pad(x, (1, 2))[..., 1:-2]       # noqa: E731  unaligned rows of an odd stride
    compare(pad(q), pad(k), pad(v), None, lengths=n, causal=True, query_start=n - Tq)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("Tq,Tk,D", [(899, 899, 64), (900, 900, 64), (70, 901, 40), (130, 1023, 64), (200, 895, 64)])
def test_key_tiles_of_both_sizes(Tq, Tk, D, kind):
    q, k, v, do = make(2, Tq, Tk, 3, 1, D, kind, seed=Tq + Tk)
    compare(q, k, v, do)
    n = torch.tensor([Tk - 3, Tk // 2], device="cuda", dtype=torch.int32)
    compare(q, k, v, do, causal=True, lengths=n, query_lengths=n.clamp(max=Tq))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Tq,Tk,D", [(150, 150, 64), (40, 60, 32), (3, 2000, 128), (150, 1000, 64)])
def test_scores_of_millions(Tq, Tk, D, kind):
    """Scores whose last bits are worth tenths: which key a row takes is up to their rounding, but what it gets lies within the
    values, and every gradient is finite."""
    from recommendsystem_amd import ops
    q, k, v, do = make(2, Tq, Tk, 4, 2, D, kind, seed=81)
    q, k = q * 1000, k * 1000
    o, lse = ops.attention_fwd(q, k, v)
    assert bool((lse > 1e5).any()) and bool(torch.isfinite(lse).all())
    hull = v.double().abs().amax(1).repeat_interleave(2, 1).unsqueeze(1)
    assert bool((o.double().abs() <= hull * (1 + 2 * torch.finfo(v.dtype).eps + (Tk + 64) * U)).all())
    for g in ops.attention_bwd(do, q, k, v, o, lse):
        assert bool(torch.isfinite(g).all())
