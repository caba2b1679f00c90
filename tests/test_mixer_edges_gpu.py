"""Operators around a recurrent mixer at the edges of their definitions: 8-bit outputs against
IEEE division, decays of long chunks, infinities at the ends of sequences and chunks and beside
padded states, calls without a sequence, and calls whose stream decides their values."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import mixer_oracle as orc

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
F8 = torch.float8_e4m3fn


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _n64(t):
    return None if t is None else t.detach().cpu().double().numpy()


# --------------------------------------------------------------------------- norm ----
@pytest.mark.parametrize("group", [None, 32, 64, 128])
@pytest.mark.parametrize("dtype,D", [(F32, 4096), (BF16, 8192), (F16, 1032), (F32, 5003), (BF16, 301),
                                     (F32, 9000), (F16, 8191)])
def test_norm_codes_are_ieee_quotients(dtype, D, group):
    """Rows of +-1 have the sum of squares D whatever its order, so the values before the 8-bit
    form are those of the 32-bit call, bit by bit; the scale is amax times the rounded 1 / 448, and
    the codes are y / scale rounded once and then to e4m3: no tolerance."""
    from pto_fuser import add_rms_norm
    for seed in range(40):
        g = _gen(seed)
        w = torch.randn(D, generator=g) * torch.exp(2 * torch.randn(D, generator=g))
        x = torch.randint(0, 2, (1, D), generator=g).mul(2).sub(1).float()
        y = add_rms_norm(x.cuda(), w.cuda())[0].cpu()
        q, _, s = add_rms_norm(x.to(dtype).cuda(), w.cuda(), out_dtype=F8, group_size=group)
        size = group or D
        parts = torch.nn.functional.pad(y, (0, -D % size)).view(1, -1, size)
        scale = torch.clamp(parts.abs().amax(-1) * torch.tensor(1 / 448.0), min=2.0 ** -126)
        want = (parts / scale[..., None]).view(1, -1)[:, :D].to(F8)
        assert torch.equal(s.cpu(), scale)
        assert torch.equal(q.cpu().float(), want.float())


@pytest.mark.parametrize("group", [None, 32, 128])
@pytest.mark.parametrize("off", [0, 1, 2])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_codes_of_values_between_two_codes(dtype, off, group):
    """Weights within a few units in the last place of the middles between two e4m3 values, times the
    scale, over rows of +-1, whose root is 1 with eps = 0 (so y is the weight): the codes are those
    of the quotient, which a product with a reciprocal misses for some. No tolerance."""
    from pto_fuser import add_rms_norm
    D = 1024
    codes = torch.arange(0, 127, dtype=torch.uint8).view(F8).float()      # 0 to 448
    middles = (codes[1:] + codes[:-1]) / 2
    size = group or D
    for seed in range(4):
        g = _gen(seed)
        amax = torch.exp(3 * torch.randn(D // size, 1, generator=g))
        scale = amax * torch.tensor(1 / 448.0)
        w = middles[torch.randint(0, len(middles), (D // size, size), generator=g)] * scale
        bits = w.view(torch.int32) + torch.randint(-2, 3, w.shape, generator=g).to(torch.int32)
        w = bits.view(F32)
        w[:, :1] = amax
        want = (w / scale).view(-1).to(F8).float()
        sign = torch.randint(0, 2, (2, D), generator=g).mul(2).sub(1).float()
        big = torch.zeros(2, D + 4, dtype=dtype, device="cuda")
        x = big[:, off:off + D]
        x.copy_(sign)
        q, _, s = add_rms_norm(x, w.view(-1).cuda(), eps=0.0, out_dtype=F8, group_size=group)
        assert torch.equal(s.cpu(), scale.view(1, -1).expand(2, -1))
        assert torch.equal(q.cpu().float(), want * sign)


def test_norm_to_8_bits_of_values_beyond_the_type():
    """An infinite value has an infinite scale: the others of its group are 0, itself NaN."""
    from pto_fuser import add_rms_norm
    for D in (256, 301):
        w = torch.ones(D)
        w[3] = 3e38
        x = torch.full((2, D), 1.0)
        x[:, 3] = 4.0               # normed to 3.9 and more, so 3e38 times it is infinite
        for group in (None, 128):
            y, _, s = add_rms_norm(x.cuda(), w.cuda(), out_dtype=F8, group_size=group)
            y, s = y.float().cpu(), s.cpu()
            assert torch.isinf(s[:, 0]).all() and torch.isnan(y[:, 3]).all()
            rest = torch.ones(D, dtype=torch.bool)
            rest[3] = False
            assert (y[:, rest][:, :100] == 0).all()


# --------------------------------------------------------------------------- scan ----
def _slots(N, T, D, n, dtype, packed=False, max_len=0):
    """Chunk slots that a call's plan takes (0: whole sequences)."""
    from pto_fuser import native as nv
    p = nv.SsmScanParams(*[8] * 14, N, T, D, n, 1, nv.dtype_code(dtype), 1, packed, 0, max_len)
    return nv.lib().ptof_ssm_scan_ws_bytes(ctypes.byref(p)) // (4 * D * (n + 1))


@pytest.mark.parametrize("T,D,S", [(65536, 2048, 2048), (65536, 4096, 4096), (262144, 2048, 8192)])
def test_scan_decay_over_long_chunks(T, D, S):
    """Without inputs the state at a chunk's first token is exp(A sum dt') h0, from the chunks'
    sums alone. Roundings, U = 2^-24 each: of a sum of 4 steps 3, of the compensated sum of
    those 2, of its addition over lanes 2, of A log2(e) 2 and of its product with the sum 1, so
    10 U of the exponent; 2^-22 for each exponential and U for each product."""
    from pto_fuser import ssm_scan
    assert _slots(1, T, D, 1, F32) == T // S
    g = _gen(S)
    dt = (0.5 + torch.rand(D, generator=g)) / S
    A = -(0.3 + 0.4 * torch.rand(D, 1, generator=g))
    zero, one = torch.zeros(1, 1, D).cuda(), torch.ones(1, 1, 1).cuda()
    y, f = ssm_scan(zero.expand(1, T, D), dt.cuda().expand(1, T, D), A.cuda(), one.expand(1, T, 1),
                    one.expand(1, T, 1), dt_softplus=False,
                    initial_state=torch.ones(1, D, 1, device="cuda"))
    j = np.arange(T // S)
    arg = (j[:, None] * S + 1.0) * (_n64(dt) * _n64(A)[:, 0])
    want = np.exp(arg)
    tol = want * (np.abs(arg) * 10 * orc.U + (j[:, None] + 1) * (2.0 ** -22 + orc.U))
    bad = ~(np.abs(_n64(y[0, ::S]) - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.abs(_n64(y[0, ::S]) / want - 1).max())


def _scan_inputs(T, D, n, dtype, seed=0):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    step = torch.exp(torch.rand(D, generator=g) * 4.6 - 9.2)
    return dict(x=r(T, D).to(dtype), dt=(0.5 * r(T, D)).to(dtype), z=r(T, D).to(dtype),
                A=-torch.arange(1, n + 1).float() * torch.exp(0.1 * r(D, n)),
                B=r(T, 1, n).to(dtype), C=r(T, 1, n).to(dtype), D=1 + 0.1 * r(D),
                bias=step + torch.log(-torch.expm1(-step)), init=r(1, D, n))


@pytest.mark.parametrize("dtype,T,D,n,slots", [(BF16, 2100, 4096, 16, 0), (BF16, 16384, 4096, 16, 16),
                                               (F16, 16384, 8192, 16, 8), (F32, 2000, 512, 16, 0),
                                               (F16, 900, 40, 24, 0)])
def test_scan_in_chunks_of_any_length_and_type(dtype, T, D, n, slots):
    """Chunks of 1024 tokens and more, and shorter ones in 16-bit types, against the oracle over
    a few of the channels (they do not meet)."""
    from pto_fuser import ssm_scan
    got = _slots(1, T, D, n, dtype)
    assert got == slots if slots else got > 1
    i = _scan_inputs(T, D, n, dtype, seed=T)
    c = {k: v.cuda() for k, v in i.items()}
    y, f = ssm_scan(c["x"][None], c["dt"][None], c["A"], c["B"][None], c["C"][None], D=c["D"],
                    z=c["z"][None], dt_bias=c["bias"], initial_state=c["init"])
    pick = torch.tensor([0, 1, D // 2 + 1, D - 1])
    at = lambda k: _n64(i[k][..., pick])
    ry, ty, rf, tf = orc.ssm_scan(at("x"), at("dt"), _n64(i["A"][pick]), _n64(i["B"]), _n64(i["C"]),
                                  [(0, T)], D=at("D"), z=at("z"), dt_bias=at("bias"),
                                  initial=_n64(i["init"][:, pick]))
    gy, gf = _n64(y[0, :, pick]), _n64(f[:, pick])
    eps, tiny = torch.finfo(dtype).eps, torch.finfo(dtype).tiny
    assert (np.abs(gf - rf) <= tf + np.abs(rf) * orc.U).all()
    assert (np.abs(gy - ry) <= ty + (np.abs(ry) + ty) * eps / 2 + tiny * eps / 2).all()


def _define(i, T, D=None, init=None, dt=None):
    """The definition in 64 bits, token by token, infinities and NaN and all. A decay below 2^-126 is
    zero in fp32 arithmetic without subnormal numbers, and zero times an infinite state is NaN:
    so it is here, where 64 bits would hold the decay (exp(dt A) for dt A < -87.3)."""
    x, B, C, A = (_n64(i[k]) for k in ("x", "B", "C", "A"))
    d = orc.softplus(_n64(i["dt"])) if dt is None else dt
    h = np.zeros(A.shape) if init is None else init.astype(np.float64)
    ys = []
    with np.errstate(all="ignore"):
        for t in range(T):
            a = np.exp(d[t][:, None] * A)
            h = np.where(a < 2.0 ** -126, 0.0, a) * h + (d[t] * x[t])[:, None] * B[t]
            ys.append((C[t] * h).sum(1) + (0.0 if D is None else D * x[t]))
    return np.stack(ys), h


def _alike(got, ref, what=""):
    """Infinities with their signs, NaN and finite values at the same places."""
    g = _n64(got)
    assert np.array_equal(np.isnan(g), np.isnan(ref)), (what, "NaN", np.argwhere(np.isnan(g) != np.isnan(ref))[:4])
    w = np.isinf(ref) | np.isinf(g)
    assert np.array_equal(np.where(w, g, 0), np.where(w, ref, 0)), (what, np.argwhere(w)[:4])


def _infinities(T, n, dtype, places, skips):
    from pto_fuser import ssm_scan
    D = 12
    for at in {T - 1, T // 2}:
        for where in places:
            i = _scan_inputs(T, D, n, dtype, seed=n)
            for k in ("B", "C"):      # of one sign: an infinite input has an infinite output
                i[k] = i[k].abs() + 0.25
            i[where][(at, 0, n - 1) if where in "BC" else (at, 3)] = float("inf")
            c = {k: v.cuda() for k, v in i.items()}
            for skip in skips:
                y, f = ssm_scan(c["x"][None], c["dt"][None], c["A"], c["B"][None], c["C"][None],
                                D=skip and c[skip])
                ry, rf = _define(i, T, D=skip and _n64(i[skip]))
                _alike(f[0], rf, (where, at, skip, "final"))
                _alike(y[0], ry, (where, at, skip, "y"))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 4, 7, 12, 16, 33, 70])
@pytest.mark.parametrize("T", [1, 16, 21, 40])
def test_scan_infinite_B_and_C(T, n, dtype):
    """An infinity in B or C at the last and at an earlier token: outputs and final state are
    infinite or NaN exactly where the definition is."""
    _infinities(T, n, dtype, ("B", "C"), (None, "D"))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 4, 7, 8, 12, 16, 33, 64, 70])
@pytest.mark.parametrize("T", [1, 16, 21, 40])
def test_scan_infinite_x_and_dt(T, n, dtype):
    """The same for x and dt, with a skip and without one (which is not a skip of zero), and with
    states that do not fill the lanes."""
    _infinities(T, n, dtype, ("x", "dt"), (None, "D"))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,D,n", [(3, 12, 8), (3, 12, 16), (2, 12, 64), (700, 1040, 16),
                                   # states that do not fill the lanes
                                   (3, 12, 1), (3, 12, 5), (2, 12, 7), (2, 12, 33), (2, 12, 70),
                                   (700, 1040, 5)])
def test_scan_step_infinities(M, D, n, dtype):
    from pto_fuser import ssm_scan_step
    for where in ("x", "dt", "B", "C", "state"):
        i = _scan_inputs(M, D, n, dtype, seed=n)
        for k in ("B", "C"):
            i[k] = i[k].abs() + 0.25
        state = torch.randn(M, D, n, generator=_gen(3))
        if where == "state":
            state[1, 3, n - 1] = float("inf")
        else:
            i[where][(1, 0, n - 1) if where in "BC" else (1, 3)] = float("inf")
        c = {k: v.cuda() for k, v in i.items()}
        for skip in (None, "D"):
            st = state.cuda()
            y = ssm_scan_step(c["x"], c["dt"], c["A"], c["B"], c["C"], st, D=skip and c[skip])
            for m in (0, 1):
                one = {k: v[m:m + 1] if k in ("x", "dt", "B", "C") else v for k, v in i.items()}
                ry, rf = _define(one, 1, D=skip and _n64(i[skip]), init=_n64(state[m]))
                _alike(st[m], rf, (where, m, skip, "state"))
                _alike(y[m:m + 1], ry, (where, m, skip, "y"))


@pytest.mark.parametrize("n", [12, 16])
def test_scan_infinities_between_chunks(n):
    """An infinite state stays infinite through chunks whose decay is below 2^-126, and a state of
    zero stays zero through chunks whose growth is beyond the type."""
    from pto_fuser import ssm_scan
    T, D = 700, 20
    assert _slots(1, T, D, n, F32) > 1
    i = _scan_inputs(T, D, n, F32, seed=1)
    i["dt"] = i["dt"].abs() + 1
    i["x"][10, 3] = float("inf")
    i["B"] = i["B"].abs() + 0.25
    c = {k: v.cuda() for k, v in i.items()}
    y, f = ssm_scan(c["x"][None], c["dt"][None], c["A"], c["B"][None], c["C"][None])
    ry, rf = _define(i, T)
    assert np.isinf(rf[3]).all()
    _alike(f[0], rf, "final")
    _alike(y[0], ry, "y")

    i = _scan_inputs(T, D, n, F32, seed=2)
    i["x"][:T - 3] = 0
    d = -_n64(i["dt"].abs() + 1) / 2       # exp(dt A) > 1 with A < 0
    c = {k: v.cuda() for k, v in i.items()}
    y, f = ssm_scan(c["x"][None], torch.tensor(d).float().cuda()[None], c["A"], c["B"][None],
                    c["C"][None], dt_softplus=False)
    ry, rf = _define(i, T, dt=torch.tensor(d).float().double().numpy())
    assert (y[0, :T - 3] == 0).all() and np.isfinite(rf).all()
    assert torch.isfinite(f).all() and torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scan_c_entry_without_a_sequence(dtype):
    """A packed call of no sequence: its tokens get zeros with zero_fill, else stay."""
    from pto_fuser import native as nv
    T, D, pitch, n = 37, 20, 23, 16
    dest = torch.full((T, pitch), 3.0, dtype=dtype, device="cuda")
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    A = torch.ones(D, n, device="cuda")
    s = [0, D] * 3 + [0, pitch] + [0, n, 0] * 2
    for fill in (0, 1):
        p = nv.SsmScanParams(*s, 0, T, D, n, 1, nv.dtype_code(dtype), 1, 1, fill, 0)
        y = dest[:, 2:2 + D]
        nv.check(nv.lib().ptof_ssm_scan_exec(
            ctypes.byref(p), None, None, nv.ptr(A), None, None, None, None, None, nv.ptr(cu), None,
            y.data_ptr(), None, None, 0, nv.stream_handle(dest.device)))
        assert (y == (0.0 if fill else 3.0)).all()
        assert (dest[:, :2] == 3.0).all() and (dest[:, 2 + D:] == 3.0).all()


# --------------------------------------------------------------------- launch plans ----
def _step_call(M=5, D=24, n=16):
    """A single-token call by its tensors, after one that left its plan."""
    from pto_fuser import ssm_scan_step
    g = _gen(7)
    r = lambda *s, dt=BF16: torch.randn(*s, generator=g).to(dt).cuda()
    a = dict(x=r(M, D), dt=r(M, D), A=-torch.rand(D, n, generator=g).cuda(), B=r(M, n), C=r(M, n),
             state=r(M, D, n, dt=F32))
    ssm_scan_step(**dict(a, state=a["state"].clone()))
    return ssm_scan_step, a


def test_a_plan_does_not_drop_tangents():
    from torch.autograd import forward_ad
    fn, a = _step_call()
    for name in a:
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                fn(**dict(a, **{name: dual}))


def test_a_plan_does_not_drop_a_sign():
    fn, a = _step_call()
    for name in a:
        with pytest.raises(ValueError, match=name + ".resolve_neg"):
            fn(**dict(a, **{name: torch._neg_view(a[name])}))


def test_a_plan_does_not_pass_a_state_that_shares_memory():
    from pto_fuser import short_conv_step, ssm_scan_step
    fn, a = _step_call()
    with pytest.raises(ValueError, match="state must not share memory"):
        fn(**dict(a, A=a["state"][1]))
    # columns of one pool: beside each other they pass, and give what they give apart
    M, D = 5, 24
    pool = torch.randn(M, 3, 3 * D, generator=_gen(1)).to(BF16).cuda()
    w = torch.randn(D, 4, generator=_gen(2)).to(BF16).cuda()
    for _ in range(3):
        x, state = pool[:, 0, D:2 * D], pool[..., :D]
        alone = state.clone(memory_format=torch.contiguous_format)
        want = short_conv_step(x.contiguous(), alone, w)
        rest = pool[..., D:].clone()
        assert torch.equal(short_conv_step(x, state, w), want)
        assert torch.equal(state, alone) and torch.equal(pool[..., D:], rest)
    with pytest.raises(ValueError, match="state must not share memory"):
        short_conv_step(pool[:, 0, D - 1:2 * D - 1], pool[..., :D], w)


def test_updates_in_place_are_seen_by_autograd():
    """A backward that saved a state or an output buffer before a call wrote into it fails, as after
    any other update in place, and does not use the new values."""
    from pto_fuser import short_conv, short_conv_step
    fn, a = _step_call()
    w4 = torch.ones(a["x"].shape[1], 4, device="cuda", dtype=BF16)
    out = torch.empty_like(a["x"])
    calls = [(a["state"], lambda: fn(**a)), (a["state"], lambda: fn(**a, out=out)),
             (out, lambda: fn(**a, out=out)), (out, lambda: short_conv(a["x"][None], w4, out=out[None]))]
    for tensor, call in calls:
        before = tensor._version
        call()
        assert tensor._version == before + 1
    weight = torch.ones(a["state"].shape[2], device="cuda", requires_grad=True)
    state = a["state"]
    loss = (state * weight).sum()
    fn(**a)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                        # no versions there, and no error
        state = torch.zeros_like(a["state"])
        for _ in range(2):
            fn(**dict(a, state=state))
            fn(**dict(a, state=state), out=torch.empty_like(a["x"]))
    conv = torch.zeros(5, 3, 24, device="cuda", dtype=BF16)
    for k in range(3):
        short_conv_step(a["x"], conv, w4)
        assert conv._version == k + 1


# ------------------------------------------------------------------------ streams ----
def test_a_call_runs_and_allocates_on_the_calling_stream():
    """The inputs of calls on a side stream are written there, behind work that takes a while, and
    results are read there, some dropped at once so that their memory is used again: a launch
    on another stream would read what is not there yet, a block of another stream's pool would
    be overwritten while it is read."""
    from pto_fuser import add_rms_norm, ssm_scan
    M, D, n = 512, 2048, 16
    g = _gen(0)
    rounds = 12
    values = torch.randn(rounds, 2, M, D, generator=g).to(BF16).cuda()
    w = torch.ones(D, device="cuda", dtype=BF16)
    A = -torch.rand(D, n, generator=g).cuda() - 0.1
    bc = torch.randn(2, 1, M, n, generator=g).to(BF16).cuda()

    def call(x):
        u = add_rms_norm(x, w)[0]
        y, f = ssm_scan(u[None], u[None], A, bc[0], bc[1])      # in chunks: it takes scratch
        return y[0], f

    assert _slots(1, M, D, n, BF16) > 1
    want = [[tuple(t.clone() for t in call(values[k, lane])) for lane in (0, 1)] for k in range(rounds)]
    lanes = [torch.cuda.current_stream(), torch.cuda.Stream()]
    xs = [torch.zeros(M, D, device="cuda", dtype=BF16) for _ in lanes]
    slow = [torch.randn(4096, 4096, device="cuda", dtype=BF16) for _ in lanes]
    got = [[None, None] for _ in range(rounds)]
    torch.cuda.synchronize()
    for k in range(rounds):
        for lane, stream in enumerate(lanes):
            with torch.cuda.stream(stream):
                for _ in range(6):
                    slow[lane] @ slow[lane]
                xs[lane].copy_(values[k, lane])
                y, f = call(xs[lane])
                got[k][lane] = (y.clone(), f.clone())
                del y, f
    torch.cuda.synchronize()
    for k in range(rounds):
        for lane in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(got[k][lane], want[k][lane])), (k, lane)
