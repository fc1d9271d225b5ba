"""Timing and accuracy cases of the sequence operators: attention over fields, click histories and cached keys (forward,
backward, single tokens), layer norm (forward, backward with the weight's and the bias's gradient, residual), and
rotary positions.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare(case, seed)` makes the inputs on
the GPU, `run(state)` is one pass: in elementary torch operations where `own` is false, through the package's operators
where it is true.  `work(case)` counts what a pass cannot do without, `exact(case, seed)` is its result in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attention(b, tq, tk, hq, hkv, d, type, causal=False, ragged=False, back=False, **name):
    return dict(name, op="attention", b=b, tq=tq, tk=tk, hq=hq, hkv=hkv, d=d, type=type, causal=causal, ragged=ragged,
                back=back)


def _norm(rows, n, type, wtype, residual=False, back=False, **name):
    return dict(name, op="norm", rows=rows, n=n, type=type, wtype=wtype, residual=residual, back=back)


def _rotary(b, t, hq, hkv, d, rot, type, interleaved, table, back=False, **name):
    return dict(name, op="rotary", b=b, t=t, hq=hq, hkv=hkv, d=d, rot=rot, type=type, interleaved=interleaved, table=table,
                back=back)


def listed():
    return [
        # a training step's interaction of the 39 fields of a 4096-sample batch: two heads of the embedding width 16
        _attention(4096, 39, 39, 2, 2, 16, "f32", back=True, name="attn fields f32 train"),
        # a training step over padded click histories of up to 200 events, every length from none on
        _attention(256, 200, 200, 8, 8, 32, "bf16", causal=True, ragged=True, back=True, name="attn histories bf16 train"),
        # pre-training over long event streams with shared key heads: the largest case
        _attention(2, 8192, 8192, 16, 4, 128, "bf16", causal=True, back=True, name="attn long bf16 train"),
        # scoring whole sessions of an odd length in one direction, half precision
        _attention(3, 1537, 1537, 12, 12, 64, "f16", name="attn sessions f16 forward"),
        # one user's next click against 333 cached events: the smallest call, where latency counts
        _attention(1, 1, 333, 4, 4, 32, "f32", ragged=True, name="attn one user f32 token"),
        # the next token of 64 users at once over caches of up to 4096 events
        _attention(64, 1, 4096, 32, 8, 128, "bf16", ragged=True, name="attn 64 users bf16 token"),
        # the norm in front of a small scoring tower
        _norm(256, 64, "f32", "f32", name="norm small f32 forward"),
        # a training step's norm over the 1024-wide first block of a 4096-sample batch
        _norm(4096, 1024, "f32", "f32", back=True, name="norm tower f32 train"),
        # a training step's residual add and norm over a long bf16 residual stream, weights kept in 32 bits
        _norm(32768, 4096, "bf16", "f32", residual=True, back=True, name="norm stream bf16 train"),
        # scoring with an odd width in half precision
        _norm(5000, 777, "f16", "f16", residual=True, name="norm odd f16 forward"),
        # positions of the next token of 64 users, far into their histories
        _rotary(64, 1, 32, 8, 128, 128, "bf16", False, 131072, name="rotary 64 users bf16 token"),
        # a training step's rotation of half of each head, neighbours paired, there and back
        _rotary(4, 4096, 32, 8, 128, 64, "bf16", True, 8192, back=True, name="rotary stream bf16 train"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm", "rotary"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "attention":
        d = rng.choice([16, 20, 24, 32, 40, 64, 80, 96, 128])
        hkv = rng.choice([1, 2, 3, 4, 8])
        hq = hkv * rng.choice([1, 1, 2, 4])
        form = rng.choice(["square", "square", "token", "chunk"])
        back = form == "square" and rng.random() < 0.6
        if form == "square":
            tq = tk = _spread(rng, 2, 3000)
        elif form == "token":
            tq, tk = 1, _spread(rng, 1, 20000)
        else:
            tq, tk = _spread(rng, 2, 300), _spread(rng, 300, 8000)
        # as many samples as fit in half of the largest listed case's products, 1024 at most
        most = int(min(1024, 2 ** 36 // (tq * tk * hq * 128), 2 ** 31 // ((tq * hq + tk * hkv) * 256)))
        return _attention(_spread(rng, 1, max(1, most)), tq, tk, hq, hkv, d, kind, causal=form != "token" and rng.random() < 0.6,
                          ragged=rng.random() < 0.5, back=back)
    if op == "norm":
        n = _spread(rng, 16, 9000)
        rows = _spread(rng, 1, min(100000, 2 ** 27 // n))
        return _norm(rows, n, kind, rng.choice([kind, "f32"]), residual=rng.random() < 0.5, back=rng.random() < 0.6)
    d = rng.choice([16, 32, 48, 64, 80, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4])
    b = _spread(rng, 1, 128)
    t = 1 if rng.random() < 0.3 else _spread(rng, 1, min(8192, 2 ** 27 // (b * (hq + hkv) * d)))
    return _rotary(b, t, hq, hkv, d, d if rng.random() < 0.5 else 2 * rng.randint(1, d // 2), kind, rng.random() < 0.5,
                   rng.choice([8192, 20000, 131072]), back=rng.random() < 0.5)


def work(case):
    e = _BYTES[case["type"]]
    if case["op"] == "attention":
        b, tq, tk, hq, hkv, d = (case[k] for k in ("b", "tq", "tk", "hq", "hkv", "d"))
        both = case["ragged"] and tq == tk                  # lengths are uniform over 0..t
        q_rows, k_rows = b * tq * (0.5 if both else 1.0), b * tk * (0.5 if case["ragged"] else 1.0)
        pairs = b * tq * tk * (1 / 3 if both else 0.5 if case["ragged"] else 1.0)
        if case["causal"]:
            pairs = pairs / 2 if tq == tk else pairs - b * tq * (tq - 1) / 2 * (0.5 if case["ragged"] else 1.0)
        qb, kb = q_rows * hq * d * e, k_rows * hkv * d * e
        return {"bytes": 2 * qb + 2 * kb + (2 * qb + 2 * kb if case["back"] else 0),
                "flops": pairs * hq * d * (14 if case["back"] else 4)}
    if case["op"] == "norm":
        x = case["rows"] * case["n"]
        tensors = 2 + (2 if case["residual"] else 0) + (2 + (1 if case["residual"] else 0) if case["back"] else 0)
        return {"bytes": tensors * x * e + case["n"] * 2 * _BYTES[case["wtype"]] * (2 if case["back"] else 1),
                "flops": x * (8 + (13 if case["back"] else 0))}
    x = case["b"] * case["t"] * (case["hq"] + case["hkv"])
    passes = 2 if case["back"] else 1
    angles = min(case["b"] * case["t"], case["table"]) * case["rot"] * 4
    return {"bytes": passes * (2 * x * case["d"] * e + angles), "flops": passes * 3 * x * case["rot"]}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]

    def normal(*shape, std=1.0, type=kind):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(type)

    s = dict(case)
    if case["op"] == "attention":
        b, tq, tk, hq, hkv, d = (case[k] for k in ("b", "tq", "tk", "hq", "hkv", "d"))
        if tq == tk and tq > 1:                             # views of one projection's output, as a layer has them
            qkv = normal(b, tq, hq + 2 * hkv, d)
            s["q"], s["k"], s["v"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:]
        else:
            s["q"], s["k"], s["v"] = normal(b, tq, hq, d), normal(b, tk, hkv, d), normal(b, tk, hkv, d)
        s["lengths"] = s["query_lengths"] = None
        if case["ragged"]:
            s["lengths"] = torch.randint(0, tk + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
            s["lengths"][0] = tk                            # the longest sample sets the padding
            s["query_lengths"] = s["lengths"] if tq == tk and tq > 1 else None
        if case["back"]:
            s["do"] = normal(b, tq, hq, d)
    elif case["op"] == "norm":
        rows, n, w = case["rows"], case["n"], _TYPES[case["wtype"]]
        s["x"] = normal(rows, n, std=2.0) + 0.5
        s["weight"], s["bias"] = 1 + normal(n, std=0.2, type=w), normal(n, std=0.2, type=w)
        s["residual"] = normal(rows, n) if case["residual"] else None
        if case["back"]:
            s["dy"] = normal(rows, n)
            s["ds"] = normal(rows, n) if case["residual"] else None
    else:
        b, t, hq, hkv, d = (case[k] for k in ("b", "t", "hq", "hkv", "d"))
        s["q"], s["k"] = normal(b, t, hq, d), normal(b, t, hkv, d)
        start = torch.randint(0, case["table"] - t + 1, (b, 1), device="cuda", generator=g)
        s["positions"] = start + torch.arange(t, device="cuda")
        freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        if own:
            from recommendsystem_amd import ops
            s["table"] = ops.RotaryTable(case["table"], case["rot"], "cuda", interleaved=case["interleaved"])
        else:
            angle = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * freq
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["back"]:
            s["dq"], s["dk"] = normal(b, t, hq, d), normal(b, t, hkv, d)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return {"attention": _run_attention, "norm": _run_norm, "rotary": _run_rotary}[s["op"]](s)


def _run_attention(s):
    if own:
        from recommendsystem_amd import ops
        how = dict(lengths=s["lengths"], query_lengths=s["query_lengths"], causal=s["causal"])
        if not s["back"]:
            return {"o": ops.attention_fwd(s["q"], s["k"], s["v"], want_lse=False, **how)[0]}
        o, lse = ops.attention_fwd(s["q"], s["k"], s["v"], **how)
        dq, dk, dv = ops.attention_bwd(s["do"], s["q"], s["k"], s["v"], o, lse, **how)
        return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    b, tq, tk, hq, hkv, d = (s[k] for k in ("b", "tq", "tk", "hq", "hkv", "d"))
    kind, scale = s["q"].dtype, d ** -0.5

    def rows(x):                                            # [b, tq, hq, d] -> [b, hkv, (hq / hkv) * tq, d], 32 bits
        return x.float().transpose(1, 2).reshape(b, hkv, hq // hkv * tq, d)

    q = rows(s["q"])
    k, v = s["k"].float().transpose(1, 2).contiguous(), s["v"].float().transpose(1, 2).contiguous()
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    hidden = _hidden(s, torch.arange(tq, device="cuda"), torch.arange(tk, device="cuda"))
    if hidden is not None:
        score.view(b, hkv, hq // hkv, tq, tk).masked_fill_(hidden.view(-1, 1, 1, *hidden.shape[1:]), -math.inf)
    top = score.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    p = p.mul_(torch.where(total > 0, 1 / total, torch.zeros_like(total)))
    o = torch.matmul(p, v)

    def heads(x):                                           # the way back, rounded to the inputs' type
        return x.view(b, hq, tq, d).transpose(1, 2).to(kind).contiguous()

    if not s["back"]:
        return {"o": heads(o)}
    lse = (total.log() + top).view(b, hq, tq)
    do = rows(s["do"])
    if s["query_lengths"] is not None:                      # rows behind a sample's last event have no part in it
        live = torch.arange(tq, device="cuda") < s["query_lengths"].view(-1, 1)
        do = (do.view(b, hq, tq, d) * live.view(b, 1, tq, 1)).view_as(do)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous()).sub_((do * o).sum(3, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    return {"o": heads(o), "lse": lse, "dq": heads(dq), "dk": dk.transpose(1, 2).to(kind).contiguous(),
            "dv": dv.transpose(1, 2).to(kind).contiguous()}


def _hidden(s, i, j):
    """Where query i does not see key j: [1 or b, tq, tk], None where all see all."""
    h = None
    if s["causal"]:
        h = (j > i.view(-1, 1) + (s["tk"] - s["tq"])).view(1, len(i), len(j))
    if s["lengths"] is not None:
        out = j.view(1, 1, -1) >= s["lengths"].view(-1, 1, 1)
        h = out.expand(-1, len(i), -1) if h is None else h | out
    if s["query_lengths"] is not None:
        h = h | (i.view(1, -1, 1) >= s["query_lengths"].view(-1, 1, 1))
    return h


def _run_norm(s):
    eps = 1e-5
    if own:
        from recommendsystem_amd import ops
        y, stream, mean, rstd = ops.layer_norm_fwd(s["x"], s["weight"], s["bias"], eps, residual=s["residual"])
        out = {"y": y} if s["residual"] is None else {"y": y, "s": stream}
        if s["back"]:
            out["dx"], out["dw"], out["db"] = ops.layer_norm_bwd(s["dy"], stream, mean, rstd, s["weight"], ds=s["ds"])
        return out
    kind, w = s["x"].dtype, s["weight"].float()
    # the residual stream is what its type holds: it is rounded before it is normalised
    stream = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(kind)
    x = stream.float()
    c = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + eps)
    xhat = c * rstd
    y = (xhat * w + s["bias"].float()).to(kind)
    out = {"y": y} if s["residual"] is None else {"y": y, "s": stream}
    if s["back"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        if s["residual"] is not None:
            dx = dx + s["ds"].float()
        out["dx"] = dx.to(kind)
        out["dw"], out["db"] = (dy * xhat).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["bias"].dtype)
    return out


def _run_rotary(s):
    if own:
        from recommendsystem_amd import ops
        q, k = ops.rotary(s["table"], s["positions"], s["q"], s["k"])
        if not s["back"]:
            return {"q": q, "k": k}
        dq, dk = ops.rotary(s["table"], s["positions"], s["dq"], s["dk"], inverse=True)
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    cos, sin = s["cos"][s["positions"]].unsqueeze(2), s["sin"][s["positions"]].unsqueeze(2)
    rot, neighbours = s["rot"], s["interleaved"]

    def turned(x, sin):
        x32 = x.float()
        a, b = (x32[..., 0:rot:2], x32[..., 1:rot:2]) if neighbours else (x32[..., :rot // 2], x32[..., rot // 2:rot])
        ra, rb = a * cos - b * sin, b * cos + a * sin
        r = torch.stack((ra, rb), -1).flatten(-2) if neighbours else torch.cat((ra, rb), -1)
        return torch.cat((r.to(x.dtype), x[..., rot:]), -1)

    out = {"q": turned(s["q"], sin), "k": turned(s["k"], sin)}
    if s["back"]:
        out["dq"], out["dk"] = turned(s["dq"], -sin), turned(s["dk"], -sin)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "norm": _exact_norm, "rotary": _exact_rotary}[case["op"]](s)


def _exact_attention(s):
    """Softmax and its derivatives by torch's own double-precision autograd, some samples and one key head at a time."""
    b, tq, tk, hq, hkv, d = (s[k] for k in ("b", "tq", "tk", "hq", "hkv", "d"))
    group = hq // hkv
    names = ("o", "lse", "dq", "dk", "dv") if s["back"] else ("o",)
    shape = {"o": (b, tq, hq, d), "lse": (b, hq, tq), "dq": (b, tq, hq, d), "dk": (b, tk, hkv, d), "dv": (b, tk, hkv, d)}
    out = {n: torch.zeros(shape[n], dtype=torch.float64, device="cuda") for n in names}
    step = max(1, 2 ** 27 // (tq * tk))
    for h in range(hkv):
        for g in range(group):
            a = h * group + g
            for n in range(0, b, step):
                c = slice(n, min(b, n + step))
                q, k, v = (x[c].double().requires_grad_(s["back"]) for x in (s["q"][:, :, a], s["k"][:, :, h], s["v"][:, :, h]))
                z = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(d)
                i, j = torch.arange(tq, device="cuda").view(1, -1, 1), torch.arange(tk, device="cuda").view(1, 1, -1)
                seen = torch.ones(1, tq, tk, dtype=torch.bool, device="cuda")
                if s["causal"]:
                    seen = seen & (j - i <= tk - tq)
                if s["lengths"] is not None:
                    seen = seen & (j < s["lengths"][c].view(-1, 1, 1))
                if s["query_lengths"] is not None:
                    seen = seen & (i < s["query_lengths"][c].view(-1, 1, 1))
                some = seen.any(2, keepdim=True)
                # a row that sees nothing is taken through a softmax of zeros and cleared after it
                w = torch.softmax(torch.where(seen, z, torch.where(some, -math.inf, 0.0).to(z)), 2) * some
                o = torch.matmul(w, v)
                out["o"][c, :, a] = o.detach()
                if s["back"]:
                    out["lse"][c, a] = torch.where(some, torch.where(seen, z, -math.inf), torch.zeros_like(z)).logsumexp(2).detach()
                    out["lse"][c, a].masked_fill_(~some.squeeze(2), -math.inf)
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"][c, :, a].double())
                    out["dq"][c, :, a] = dq
                    out["dk"][c, :, h] += dk
                    out["dv"][c, :, h] += dv
    return out


def _exact_norm(s):
    kind = s["x"].dtype
    x = s["x"].double() if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(kind).double()
    out = {} if s["residual"] is None else {"s": x.clone()}
    if not s["back"]:
        out["y"] = torch.empty_like(x)
    rows, n = x.shape
    w, bias = s["weight"].double(), s["bias"].double()
    step = max(1, 2 ** 27 // n)
    parts = []
    for r in range(0, rows, step):
        z = x[r:r + step]
        var, mean = torch.var_mean(z, 1, correction=0, keepdim=True)
        sd = torch.sqrt(var + 1e-5)
        unit = (z - mean) / sd
        if not s["back"]:
            out["y"][r:r + step] = unit * w + bias
            continue
        dy = s["dy"][r:r + step].double()
        dunit = dy * w
        # through the standard deviation and the mean, one after the other
        dsd = -(dunit * unit).sum(1, keepdim=True) / sd
        dc = dunit / sd + dsd * unit / n
        dx = dc - dc.sum(1, keepdim=True) / n
        if s["residual"] is not None:
            dx = dx + s["ds"][r:r + step].double()
        parts.append((unit * w + bias, dx, (dy * unit).sum(0), dy.sum(0)))
    if s["back"]:
        out["y"], out["dx"] = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
        out["dw"], out["db"] = torch.stack([p[2] for p in parts]).sum(0), torch.stack([p[3] for p in parts]).sum(0)
    return out


def _exact_rotary(s):
    """Pairs as complex numbers, times exp(i angle)."""
    rot = s["rot"]
    turns = s["positions"].double().unsqueeze(-1) * torch.exp(
        torch.arange(rot // 2, device="cuda", dtype=torch.float64) * (-2 * math.log(10000.0) / rot))
    unit = torch.polar(torch.ones_like(turns), turns).unsqueeze(2)

    def turned(x, by):
        y = x.double()
        a = y[..., :rot]
        pairs = a.unflatten(-1, (rot // 2, 2)) if s["interleaved"] else a.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        z = z if s["interleaved"] else z.transpose(-1, -2)
        return torch.cat((z.flatten(-2), y[..., rot:]), -1)

    out = {"q": turned(s["q"], unit), "k": turned(s["k"], unit)}
    if s["back"]:
        out["dq"], out["dk"] = turned(s["dq"], unit.conj()), turned(s["dk"], unit.conj())
    return out
