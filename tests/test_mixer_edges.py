"""Arguments of the operators around a recurrent mixer that are refused although their shapes and
types are right, checked before anything touches a device."""
import pytest
import torch
from torch.autograd import forward_ad

import pto_fuser as pf

F32, BF16 = torch.float32, torch.bfloat16


def z(*s, dtype=BF16):
    return torch.zeros(*s, dtype=dtype)


def _calls():
    """Each entry point with its tensors by name."""
    A, st = z(8, 4, dtype=F32), z(4, 8, 4, dtype=F32)
    return {
        pf.short_conv: dict(x=z(2, 5, 8), weight=z(8, 4), bias=z(8), initial_state=z(2, 3, 8)),
        pf.short_conv_step: dict(x=z(3, 8), state=z(4, 3, 8), weight=z(8, 4), bias=z(8)),
        pf.ssm_scan: dict(x=z(2, 5, 8), dt=z(2, 5, 8), A=A, B=z(2, 5, 4), C=z(2, 5, 4),
                          D=z(8, dtype=F32), z=z(2, 5, 8), dt_bias=z(8, dtype=F32),
                          initial_state=z(2, 8, 4, dtype=F32)),
        pf.ssm_scan_step: dict(x=z(3, 8), dt=z(3, 8), A=A, B=z(3, 4), C=z(3, 4), state=st,
                               D=z(8, dtype=F32), z=z(3, 8), dt_bias=z(8, dtype=F32)),
        pf.add_rms_norm: dict(x=z(3, 8), weight=z(8), residual=z(3, 8)),
    }


CASES = [(f, k) for f, a in _calls().items() for k in a]


@pytest.mark.parametrize("fn,name", CASES, ids=[f"{f.__name__}-{k}" for f, k in CASES])
def test_forward_mode_tangents_are_refused(fn, name):
    a = _calls()[fn]
    with forward_ad.dual_level():
        a[name] = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            fn(**a)
        with torch.no_grad(), pytest.raises(ValueError, match="no forward-mode derivative"):
            fn(**a)         # no_grad stops the backward only
        with torch.inference_mode(), pytest.raises(ValueError, match="CUDA tensors"):
            fn(**a)
    with pytest.raises(ValueError, match="no forward-mode derivative"):
        torch.func.jvp(lambda t: fn(**dict(a, **{name: t})), (_calls()[fn][name],),
                       (torch.ones_like(a[name]),))


@pytest.mark.parametrize("fn,name", CASES, ids=[f"{f.__name__}-{k}" for f, k in CASES])
def test_negated_views_are_refused(fn, name):
    """The memory of such a view holds the values before the sign."""
    a = _calls()[fn]
    a[name] = torch._neg_view(a[name])
    with pytest.raises(ValueError, match=name + ".resolve_neg"):
        fn(**a)
    a[name] = a[name].resolve_neg()
    with pytest.raises(ValueError, match="CUDA tensors"):
        fn(**a)


def test_a_state_that_shares_memory_with_an_input_is_refused():
    """It is written while other blocks may still read: a race, whatever the order of the rows."""
    def refused(fn, a, **over):
        with pytest.raises(ValueError, match="state must not share memory"):
            fn(**dict(a, **over))
    a = _calls()[pf.short_conv_step]
    st = a["state"]
    refused(pf.short_conv_step, a, x=st[:3, 1])
    refused(pf.short_conv_step, a, x=st[:3, 2], slots=z(3, dtype=torch.int32))
    refused(pf.short_conv_step, a, weight=st.view(-1)[:32].view(8, 4))
    refused(pf.short_conv_step, a, bias=st[3, 2])
    a = _calls()[pf.ssm_scan_step]
    refused(pf.ssm_scan_step, a, A=a["state"][1])
    refused(pf.ssm_scan_step, a, D=a["state"].view(-1)[8:16])
    f = {k: v.float() for k, v in a.items()}
    refused(pf.ssm_scan_step, f, x=f["state"][:3, :, 0].contiguous(), z=f["state"][0].view(4, 8)[:3])
    slots = z(128, dtype=torch.int32)
    refused(pf.ssm_scan_step, f, slots=slots[:3], state=slots.view(F32).view(4, 8, 4))
    pool = z(4, 3, 20)           # columns of one pool, side by side, are apart
    with pytest.raises(ValueError, match="CUDA tensors"):
        pf.short_conv_step(pool[:3, 0, 8:16], pool[..., :8], z(8, 4))


def test_values_of_eps_are_not_collected():
    """Values that never come again, and such as are refused, leave nothing that grows."""
    from pto_fuser import mixer
    x, w = z(3, 8), z(8)
    for k in range(3000):
        with pytest.raises(ValueError, match="CUDA tensors"):
            pf.add_rms_norm(x, w, eps=1e-6 * (k + 1))
        with pytest.raises(ValueError, match="eps"):
            pf.add_rms_norm(x, w, eps=float("nan"))
        with pytest.raises(ValueError, match="eps"):
            pf.add_rms_norm(x, w, eps=-1.0 - k)
    assert len(mixer._EPS) <= 1000
    numbers = list(mixer._EPS.values())
    assert len(set(numbers)) == len(numbers)


def test_a_launch_module_that_cannot_be_loaded_is_not_called_missing(monkeypatch, tmp_path):
    import sys

    from pto_fuser import _native, native
    native.launcher()
    monkeypatch.setattr(native, "_launcher", None)
    monkeypatch.delattr(_native, "_launch")
    monkeypatch.setitem(sys.modules, "pto_fuser._native._launch", None)     # its import fails
    with pytest.raises(RuntimeError, match="built for another torch or Python"):
        native.launcher()
    monkeypatch.setattr(native, "LIB_PATH", str(tmp_path / "lib.so"))
    with pytest.raises(RuntimeError, match="is missing"):
        native.launcher()
