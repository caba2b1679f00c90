"""Measured cases of the operators around a recurrent token mixer: the short causal convolution
in front of it, the selective state space scan, and the root-mean-square norm with the
residual's addition.

Each operator has its form for prompts and, where it keeps a state, its form for single tokens.
``run`` computes the plain form in elementary torch operations, or calls the framework's
kernels where ``own`` is true; ``exact`` restates the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_FP8_MAX = 448.0          # largest finite e4m3 value
_TINY = 2.0 ** -126       # smallest normal fp32: floor of an 8-bit scale


# ------------------------------------------------------------------------ cases ----
def listed():
    return [
        # decode of a few sequences: q, k, v channels of 32 heads of 128 share one convolution
        dict(name="conv step 8x12288", op="conv_step", dtype="bf16", rows=8, slots=16,
             channels=12288, width=4),
        # a packed prefill batch with chunked prompts: sequences that continue from a state,
        # one of a single token and an empty one
        dict(name="conv packed 5640x8192", op="conv", dtype="bf16", channels=8192, width=4,
             lengths="2048,1,77,0,3001,513", packed=True, initial=True),
        # the longest prompt of the forward's own configurations, all q, k, v channels
        dict(name="conv prompt 16384x12288", op="conv", dtype="bf16", channels=12288, width=4,
             lengths="16384", packed=False, initial=False),
        # decode of one sequence: latency
        dict(name="scan step 1x4096", op="scan_step", dtype="bf16", rows=1, slots=4,
             channels=4096, states=16, groups=1),
        # decode of a full serving batch: the states' traffic
        dict(name="scan step 512x8192", op="scan_step", dtype="bf16", rows=512, slots=640,
             channels=8192, states=16, groups=1),
        # one long prompt: few rows, a long axis
        dict(name="scan prompt 16384x4096", op="scan", dtype="bf16", channels=4096, states=16,
             groups=1, lengths="16384", packed=False, initial=False),
        # a batch of equal prompts: work for every SM
        dict(name="scan batch 8x2048x5120", op="scan", dtype="bf16", channels=5120, states=16,
             groups=1, lengths="2048,2048,2048,2048,2048,2048,2048,2048", packed=False,
             initial=False),
        # a ragged packed batch with an odd channel count, continuing from states
        dict(name="scan packed 2999x1802", op="scan", dtype="f16", channels=1802, states=16,
             groups=1, lengths="1500,1,63,0,700,735", packed=True, initial=True),
        # full precision, grouped B and C and a wide state
        dict(name="scan f32 777x512 n64", op="scan", dtype="f32", channels=512, states=64,
             groups=4, lengths="777", packed=False, initial=True),
        # decode of one sequence: norm before a product in 8 bits with one scale a token
        dict(name="norm 1x4096 e4m3", op="norm", dtype="bf16", rows=1, columns=4096,
             residual="bf16", quant="token", group=0),
        # a prefill batch: norm before a product in 8 bits with a scale for 128 columns
        dict(name="norm 16384x8192 e4m3", op="norm", dtype="bf16", rows=16384, columns=8192,
             residual="bf16", quant="group", group=128),
        # odd rows and columns, an fp32 residual stream, no 8-bit output
        dict(name="norm 3001x5003", op="norm", dtype="f16", rows=3001, columns=5003,
             residual="f32", quant="none", group=0),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cut(rng, total, parts):
    """`total` tokens in `parts` sequences, empty ones and single tokens among them."""
    at = sorted(rng.randint(0, total) for _ in range(parts - 1))
    return ",".join(str(b - a) for a, b in zip([0] + at, at + [total]))


def _draw_lengths(rng, most):
    total = _log_int(rng, 1, most)
    if rng.random() < 0.5:
        return dict(lengths=_cut(rng, total, rng.randint(1, 12)), packed=True,
                    initial=rng.random() < 0.7)
    batch = rng.randint(1, min(8, total))
    return dict(lengths=",".join([str(total // batch)] * batch), packed=False,
                initial=rng.random() < 0.5)


def draw(rng):
    op = rng.choice(["conv", "conv_step", "scan", "scan", "scan_step", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "conv":
        d = _log_int(rng, 64, 12288)
        d -= d % 8 if rng.random() < 0.6 else 0
        return dict(op=op, dtype=dtype, channels=d, width=rng.randint(2, 4),
                    **_draw_lengths(rng, 8192))
    if op == "conv_step":
        rows = _log_int(rng, 1, 512)
        d = _log_int(rng, 64, 12288)
        d -= d % 8 if rng.random() < 0.6 else 0
        return dict(op=op, dtype=dtype, rows=rows, slots=rows + rng.randint(0, 64), channels=d,
                    width=rng.randint(2, 4))
    if op == "scan":
        groups = rng.choice([1, 1, 1, 2, 4])
        n = rng.choice([16, 16, 16, 8, 32, 64, rng.randint(1, 64)])
        d = groups * _log_int(rng, 16, 8192 // groups)
        most = max(1, min(16384, int(1e9) // (d * n)))
        return dict(op=op, dtype=dtype, channels=d, states=n, groups=groups,
                    **_draw_lengths(rng, most))
    if op == "scan_step":
        groups = rng.choice([1, 1, 1, 2, 4])
        n = rng.choice([16, 16, 16, 8, 32, 64, rng.randint(1, 64)])
        rows = _log_int(rng, 1, 512)
        d = groups * _log_int(rng, 16, max(17, min(8192, 512 * 8192 * 16 // (rows * n)) // groups))
        return dict(op=op, dtype=dtype, rows=rows, slots=rows + rng.randint(0, 64), channels=d,
                    states=n, groups=groups)
    cols = _log_int(rng, 64, 16384)
    cols -= cols % 8 if rng.random() < 0.6 else 0
    quant = rng.choice(["none", "token", "group"])
    return dict(op=op, dtype=dtype, rows=_log_int(rng, 1, min(16384, (1 << 26) // cols)),
                columns=cols, residual=rng.choice(["none", dtype, "f32"]), quant=quant,
                group=rng.choice([32, 64, 128]) if quant == "group" else 0)


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


# ----------------------------------------------------------------------- inputs ----
def _prepare_tokens(case, s, gen, dt):
    """Where the sequences of a prompt case lie: cu_seqlens for a packed batch, and for both
    forms the index tensors that the plain forms gather by."""
    lens = _lengths(case)
    starts = [sum(lens[:i]) for i in range(len(lens))]
    full = [i for i, n in enumerate(lens) if n]
    total = sum(lens)
    dev = lambda v, t=torch.int64: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    s["total"], s["seqs"] = total, len(lens)
    s["shape"] = (total,) if case["packed"] else (len(lens), lens[0])
    s["cu"] = dev(starts + [total], torch.int32) if case["packed"] else None
    s["max_len"] = max(lens)
    s["seq_of"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), dev(lens))
    s["start_of"] = dev(starts)[s["seq_of"]]
    s["full"], s["first"] = dev(full), dev([starts[i] for i in full])
    s["last"] = dev([starts[i] + lens[i] - 1 for i in full])


def _mixer_weights(case, s, gen):
    """A, D, dt_bias of a selective layer: A near -(1 .. n), steps log-uniform in [1e-3, 1e-1]."""
    d, n = case["channels"], case["states"]
    rnd = lambda *sh: torch.randn(*sh, generator=gen, device="cuda")  # noqa: E731
    s["A"] = -torch.arange(1, n + 1, device="cuda", dtype=torch.float32) * torch.exp(0.1 * rnd(d, n))
    s["D"] = 1.0 + 0.1 * rnd(d)
    step = torch.exp(torch.rand(d, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rnd = lambda *sh: torch.randn(*sh, generator=gen, device="cuda")  # noqa: E731
    t = _TYPES[case["dtype"]]
    s = {"case": dict(case)}
    op = case["op"]
    if op in ("conv", "conv_step"):
        d, w = case["channels"], case["width"]
        s["weight"] = (rnd(d, w) * w ** -0.5).to(t)
        s["bias"] = (0.1 * rnd(d)).to(t)
        if op == "conv":
            _prepare_tokens(case, s, gen, t)
            s["x"] = rnd(*s["shape"], d).to(t)
            s["initial"] = rnd(s["seqs"], w - 1, d).to(t) if case["initial"] else None
        else:
            s["x"] = rnd(case["rows"], d).to(t)
            s["state"] = rnd(case["slots"], w - 1, d).to(t)
            s["at"] = torch.randperm(case["slots"], generator=gen, device="cuda")[:case["rows"]]
            s["at"] = s["at"].to(torch.int32)
        return s
    if op in ("scan", "scan_step"):
        d, n, g = case["channels"], case["states"], case["groups"]
        _mixer_weights(case, s, gen)
        if op == "scan":
            _prepare_tokens(case, s, gen, t)
            shape = s["shape"]
            s["initial"] = rnd(s["seqs"], d, n) if case["initial"] else None
        else:
            shape = (case["rows"],)
            s["state"] = rnd(case["slots"], d, n)
            s["at"] = torch.randperm(case["slots"], generator=gen, device="cuda")[:case["rows"]]
            s["at"] = s["at"].to(torch.int32)
        # x and z are the halves of one projection, B and C of another, as a layer has them
        xz = rnd(*shape, 2 * d).to(t)
        bc = rnd(*shape, 2 * g * n).to(t)
        s["x"], s["z"] = xz[..., :d], xz[..., d:]
        s["B"] = bc[..., :g * n].unflatten(-1, (g, n))
        s["C"] = bc[..., g * n:].unflatten(-1, (g, n))
        s["dt"] = (0.5 * rnd(*shape, d)).to(t)
        return s
    m, d = case["rows"], case["columns"]
    s["x"] = rnd(m, d).to(t)
    s["residual"] = None
    if case["residual"] != "none":
        s["residual"] = (4.0 * rnd(m, d)).to(_TYPES[case["residual"]])
    s["weight"] = (1.0 + 0.1 * rnd(d)).to(t)
    return s


# ------------------------------------------------------------------ plain forms ----
def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _softplus(v):
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-torch.abs(v)))


def _plain_conv(s):
    x = s["x"].reshape(s["total"], -1).float()
    w, b = s["weight"].float(), s["bias"].float()
    d, k = w.shape
    if s["initial"] is None:
        past = torch.zeros(s["seqs"] * (k - 1), d, device=x.device)
    else:
        past = s["initial"].float().reshape(-1, d)
    source = torch.cat([x, past])

    def rows(token, seq, first):
        """Rows of `source` that hold the inputs at `token` of the sequences `seq`."""
        before = s["total"] + seq * (k - 1) + (k - 1) + token - first
        return torch.where(token >= first, token, before)

    t = torch.arange(s["total"], device=x.device)[:, None] + torch.arange(1 - k, 1, device=x.device)
    y = (source[rows(t, s["seq_of"][:, None], s["start_of"][:, None])] * w.t()).sum(1) + b
    final = past.reshape(s["seqs"], k - 1, d).clone()
    t = s["last"][:, None] + torch.arange(2 - k, 1, device=x.device)
    final[s["full"]] = source[rows(t, s["full"][:, None], s["first"][:, None])]
    return _silu(y).to(s["x"].dtype).reshape(s["x"].shape), final.to(s["x"].dtype)


def _plain_conv_step(s):
    at = s["at"].long()
    window = torch.cat([s["state"][at], s["x"][:, None]], 1)
    y = (window.float() * s["weight"].float().t()).sum(1) + s["bias"].float()
    s["state"][at] = window[:, 1:]
    return _silu(y).to(s["x"].dtype)


def _linear_scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] with h[-1] = 0 along the first axis: neighbours are joined,
    the half as long scan gives every second value, and one step the others."""
    t = a.shape[0]
    if t == 1:
        return b
    e = t - t % 2
    half = _linear_scan(a[1:e:2] * a[0:e:2], a[1:e:2] * b[0:e:2] + b[1:e:2])
    h = torch.empty_like(b)
    h[1:e:2] = half
    h[0] = b[0]
    h[2::2] = a[2::2] * half[:(t - 1) // 2] + b[2::2]
    return h


def _per_channel(v, d):
    """[.., groups, n] -> [.., channels or 1, n]"""
    return v if v.shape[-2] == 1 else v.repeat_interleave(d // v.shape[-2], -2)


def _plain_scan(s):
    d, n = s["A"].shape
    x, z = (s[k].reshape(-1, d).float() for k in ("x", "z"))
    b, c = (s[k].reshape(s["total"], -1, n).float() for k in ("B", "C"))
    dt = _softplus(s["dt"].reshape(-1, d).float() + s["dt_bias"])
    decay = torch.exp(dt[:, :, None] * s["A"])
    add = (dt * x)[:, :, None] * _per_channel(b, d)
    if s["initial"] is not None:
        add[s["first"]] += decay[s["first"]] * s["initial"][s["full"]]
    decay[s["first"]] = 0.0
    h = _linear_scan(decay, add)
    del decay, add
    y = (h * _per_channel(c, d)).sum(-1) + s["D"] * x
    if s["initial"] is None:
        final = torch.zeros(s["seqs"], d, n, device=x.device)
    else:
        final = s["initial"].clone()
    final[s["full"]] = h[s["last"]]
    return (y * _silu(z)).to(s["x"].dtype).reshape(s["x"].shape), final


def _plain_scan_step(s):
    d = s["A"].shape[0]
    at = s["at"].long()
    x, z = s["x"].float(), s["z"].float()
    dt = _softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(dt[:, :, None] * s["A"]) * s["state"][at]
    h = h + (dt * x)[:, :, None] * _per_channel(s["B"].float(), d)
    s["state"][at] = h
    y = (h * _per_channel(s["C"].float(), d)).sum(-1) + s["D"] * x
    return (y * _silu(z)).to(s["x"].dtype)


def _grouped(y, group):
    """[m, d] -> [m, groups, columns of a group], zeros behind the last column."""
    d = y.shape[1]
    group = group or d
    y = torch.nn.functional.pad(y, (0, -d % group))
    return y.reshape(y.shape[0], -1, group)


def _plain_norm(s):
    case = s["case"]
    h = s["x"].float()
    out = {}
    if s["residual"] is not None:
        h = h + s["residual"].float()
        out["residual"] = h.to(s["residual"].dtype)
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    if case["quant"] == "none":
        out["y"] = y.to(s["x"].dtype)
        return out
    y = _grouped(y, case["group"])
    scale = torch.clamp(y.abs().amax(-1) / _FP8_MAX, min=_TINY)
    q = torch.clamp(y / scale[:, :, None], -_FP8_MAX, _FP8_MAX)
    out["y"] = q.reshape(q.shape[0], -1)[:, :case["columns"]].to(torch.float8_e4m3fn)
    out["scale"] = scale
    return out


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "pto-fuser_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import pto_fuser
    return pto_fuser


def run(s):
    op = s["case"]["op"]
    if own:
        f = _framework()
        if op == "conv":
            y, final = f.short_conv(s["x"], s["weight"], s["bias"], activation="silu",
                                    initial_state=s["initial"], cu_seqlens=s["cu"])
            return {"y": y, "final": final}
        if op == "conv_step":
            y = f.short_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu",
                                  slots=s["at"])
            return {"y": y, "state": s["state"]}
        if op == "scan":
            y, final = f.ssm_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                  dt_bias=s["dt_bias"], dt_softplus=True,
                                  initial_state=s["initial"], cu_seqlens=s["cu"],
                                  max_seqlen=s["max_len"])
            return {"y": y, "final": final}
        if op == "scan_step":
            y = f.ssm_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"],
                                z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True, slots=s["at"])
            return {"y": y, "state": s["state"]}
        quant = s["case"]["quant"]
        y, residual, scale = f.add_rms_norm(
            s["x"], s["weight"], s["residual"], eps=1e-6,
            out_dtype=None if quant == "none" else torch.float8_e4m3fn,
            group_size=s["case"]["group"] or None)
        out = {"y": y}
        if residual is not None:
            out["residual"] = residual
        if scale is not None:
            out["scale"] = scale
        return out
    if op == "conv":
        y, final = _plain_conv(s)
        return {"y": y, "final": final}
    if op == "conv_step":
        return {"y": _plain_conv_step(s), "state": s["state"]}
    if op == "scan":
        y, final = _plain_scan(s)
        return {"y": y, "final": final}
    if op == "scan_step":
        return {"y": _plain_scan_step(s), "state": s["state"]}
    return _plain_norm(s)


# ------------------------------------------------------------------------- work ----
def work(case):
    e = {"bf16": 2, "f16": 2, "f32": 4}
    op, k = case["op"], e[case["dtype"]]
    if op in ("conv", "conv_step"):
        d, w = case["channels"], case["width"]
        weights = d * (w + 1) * k
        if op == "conv":
            lens = _lengths(case)
            m, rows = sum(lens), len(lens)
            past = rows * (w - 1) * d * k
            moved = 2 * m * d * k + past * (2 if case["initial"] else 1)
            moved += 4 * (rows + 1) if case["packed"] else 0
        else:
            m = case["rows"]
            moved = 2 * m * d * k + 2 * m * (w - 1) * d * k + 4 * m
        return {"bytes": moved + weights, "flops": m * d * (2 * w + 5)}
    if op in ("scan", "scan_step"):
        d, n, g = case["channels"], case["states"], case["groups"]
        weights = 4 * d * n + 8 * d
        if op == "scan":
            lens = _lengths(case)
            m, rows = sum(lens), len(lens)
            state = 4 * rows * d * n * (2 if case["initial"] else 1)
            state += 4 * (rows + 1) if case["packed"] else 0
        else:
            m = case["rows"]
            state = 8 * m * d * n + 4 * m
        return {"bytes": m * (4 * d + 2 * g * n) * k + state + weights,
                "flops": m * d * (7 * n + 14)}
    m, d = case["rows"], case["columns"]
    moved = m * d * k + d * k + m * d * (1 if case["quant"] != "none" else k)
    if case["residual"] != "none":
        moved += 2 * m * d * e[case["residual"]]
    if case["quant"] != "none":
        moved += 4 * m * -(-d // (case["group"] or d))
    return {"bytes": moved, "flops": m * d * 6}


# ------------------------------------------------------------------------ exact ----
def _exact_conv(s):
    """Each sequence on its own: its past in front, one shifted product a tap."""
    x = s["x"].reshape(s["total"], -1).double()
    w = s["weight"].double()
    d, k = w.shape
    y, final, at = torch.empty_like(x), [], 0
    for i, n in enumerate(_lengths(s["case"])):
        past = x.new_zeros(k - 1, d) if s["initial"] is None else s["initial"][i].double()
        line = torch.cat([past, x[at:at + n]])
        v = s["bias"].double().expand(n, d)
        for j in range(k):
            v = v + w[:, j] * line[j:j + n]
        y[at:at + n] = v * torch.sigmoid(v)
        final.append(line[n:])
        at += n
    return {"y": y.reshape(s["x"].shape), "final": torch.stack(final)}


def _exact_scan(s):
    """The recurrence as it is written, token after token."""
    a = s["A"].double()
    d, n = a.shape
    x, z, dt = (s[k].reshape(-1, d).double() for k in ("x", "z", "dt"))
    per = d // s["B"].shape[-2]
    b, c = (s[k].reshape(s["total"], -1, n).double() for k in ("B", "C"))
    dt = dt + s["dt_bias"].double()
    dt = torch.where(dt > 30, dt, torch.log1p(torch.exp(torch.clamp(dt, max=30.0))))
    y, final, at = torch.empty_like(x), [], 0
    for i, length in enumerate(_lengths(s["case"])):
        h = x.new_zeros(d, n) if s["initial"] is None else s["initial"][i].double()
        for t in range(at, at + length):
            bt = b[t].repeat_interleave(per, 0)
            h = torch.exp(dt[t][:, None] * a) * h + (dt[t] * x[t])[:, None] * bt
            y[t] = (h * c[t].repeat_interleave(per, 0)).sum(1)
        final.append(h)
        at += length
    y = (y + s["D"].double() * x) * z * torch.sigmoid(z)
    return {"y": y.reshape(s["x"].shape), "final": torch.stack(final)}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "conv":
        return _exact_conv(s)
    if op == "scan":
        return _exact_scan(s)
    if op == "conv_step":
        at = s["at"].long()
        state = s["state"].double()
        v = s["x"].double() * s["weight"][:, -1].double() + s["bias"].double()
        for j in range(case["width"] - 1):
            v = v + state[at, j] * s["weight"][:, j].double()
        state[at] = torch.cat([state[at, 1:], s["x"].double()[:, None]], 1)
        return {"y": v * torch.sigmoid(v), "state": state}
    if op == "scan_step":
        at = s["at"].long()
        per = case["channels"] // case["groups"]
        dt = s["dt"].double() + s["dt_bias"].double()
        dt = torch.where(dt > 30, dt, torch.log1p(torch.exp(torch.clamp(dt, max=30.0))))
        x, z, state = s["x"].double(), s["z"].double(), s["state"].double()
        y = s["D"].double() * x
        for j in range(case["states"]):
            h = state[at, :, j] * torch.exp(dt * s["A"][:, j].double())
            h = h + dt * x * s["B"][:, :, j].double().repeat_interleave(per, 1)
            y = y + h * s["C"][:, :, j].double().repeat_interleave(per, 1)
            state[at, :, j] = h
        return {"y": y * z * torch.sigmoid(z), "state": state}
    h = s["x"].double()
    out = {}
    if s["residual"] is not None:
        h = h + s["residual"].double()
        out["residual"] = h
    y = h / torch.sqrt(h.square().sum(1, keepdim=True) / h.shape[1] + 1e-6) * s["weight"].double()
    if case["quant"] == "none":
        out["y"] = y
        return out
    group = case["group"] or case["columns"]
    most = [p.abs().max(1).values for p in y.split(group, 1)]
    scale = torch.stack(most, 1) / _FP8_MAX
    parts = [p / scale[:, i:i + 1] for i, p in enumerate(y.split(group, 1))]
    out["y"], out["scale"] = torch.cat(parts, 1), scale
    return out
