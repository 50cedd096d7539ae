"""The 64-bit formulas the GPU tests compare against, checked on the CPU: against autograd of the plain
recurrence and against differences; and the refusals of the C entry points, which need no device."""
import ctypes

import pytest
import torch

from fm_b200 import capi
from tests import ssm_ref as R

F64 = torch.float64


def scan_inputs(Bn=2, D=4, T=11, N=3, G=2, lengths=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, dtype=F64)
    i = dict(x=n(Bn, D, T), delta=n(Bn, D, T), A=-torch.rand(D, N, generator=g, dtype=F64) * 2, B=n(Bn, G, N, T), C=n(Bn, G, N, T),
             D=n(D), z=n(Bn, D, T), delta_bias=n(D), h0=n(Bn, D, N), lengths=lengths)
    return i, (n(Bn, D, T), n(Bn, D, N))


def autograd_ssm(i, softplus_on):
    """The recurrence with torch ops autograd can follow; returns (y, last)."""
    dt = i["delta"] + i["delta_bias"][:, None]
    dt = torch.nn.functional.softplus(dt, threshold=100) if softplus_on else dt
    per = i["x"].shape[1] // i["B"].shape[1]
    h, ys = i["h0"], []
    T = i["x"].shape[-1]
    n = i["lengths"] if i["lengths"] is not None else torch.full((i["x"].shape[0],), T)
    for t in range(T):
        on = (t < n)[:, None, None]
        d = dt[:, :, t, None]
        new = torch.exp(d * i["A"]) * h + d * i["B"][..., t].repeat_interleave(per, 1) * i["x"][:, :, t, None]
        h = torch.where(on, new, h)
        y = (h * i["C"][..., t].repeat_interleave(per, 1)).sum(-1) + i["D"] * i["x"][..., t]
        ys.append(torch.where(on[..., 0], y * torch.nn.functional.silu(i["z"][..., t]), torch.zeros_like(y)))
    return torch.stack(ys, -1), h


@pytest.mark.parametrize("softplus_on", [False, True])
@pytest.mark.parametrize("lengths", [None, [11, 4], [0, 7]])
def test_scan_formula_equals_autograd(softplus_on, lengths):
    i, grads = scan_inputs(lengths=None if lengths is None else torch.tensor(lengths))
    if not softplus_on:
        i["delta"] = i["delta"].abs()
    leaves = {k: v.clone().requires_grad_(True) for k, v in i.items() if k != "lengths"}
    y, last = autograd_ssm({**leaves, "lengths": i["lengths"]}, softplus_on)
    got = torch.autograd.grad((y, last), list(leaves.values()), grads)
    ref = R.ssm(i, softplus_on, grads)
    torch.testing.assert_close(ref["y"], y.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(ref["last"], last.detach(), rtol=1e-12, atol=1e-12)
    for name, v in zip(leaves, got):
        torch.testing.assert_close(ref["d" + name], v, rtol=1e-11, atol=1e-11, msg=name)


def test_scan_formula_against_differences():
    i, grads = scan_inputs(seed=3)
    ref = R.ssm(i, True, grads)
    g = torch.Generator().manual_seed(9)
    f = lambda j: sum((a * b).sum() for a, b in zip(grads, (lambda r: (r["y"], r["last"]))(R.ssm(j, True))))
    for k in ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0"):
        v, e = torch.randn(i[k].shape, generator=g, dtype=F64), 1e-6
        num = (f({**i, k: i[k] + e * v}) - f({**i, k: i[k] - e * v})) / (2 * e)
        torch.testing.assert_close((ref["d" + k] * v).sum(), num, rtol=1e-7, atol=1e-7, msg=k)


@pytest.mark.parametrize("silu_on", [False, True])
@pytest.mark.parametrize("lengths", [None, [9, 2], [0, 1]])
@pytest.mark.parametrize("K", [2, 4, 8])
def test_filter_formula_equals_autograd(silu_on, lengths, K):
    g = torch.Generator().manual_seed(K)
    n = lambda *s: torch.randn(*s, generator=g, dtype=F64)
    Bn, D, T = 2, 3, 9
    i = dict(x=n(Bn, D, T), w=n(D, K), b=n(D), x0=n(Bn, D, K - 1))
    grads = (n(Bn, D, T), n(Bn, D, K - 1))
    leaves = {k: v.clone().requires_grad_(True) for k, v in i.items()}
    ends = [T, T] if lengths is None else lengths
    live = R.live_mask(None if lengths is None else torch.tensor(lengths), Bn, T)[:, None]
    ext = torch.cat([leaves["x0"], leaves["x"]], -1)
    y = torch.nn.functional.conv1d(ext, leaves["w"][:, None], leaves["b"], groups=D)
    y = torch.nn.functional.silu(y) if silu_on else y
    last = torch.stack([ext[k, :, e:e + K - 1] for k, e in enumerate(ends)])
    y = torch.where(live, y, torch.zeros_like(y))
    got = torch.autograd.grad((y, last), list(leaves.values()), grads)
    ref = R.conv({**i, "lengths": None if lengths is None else torch.tensor(lengths)}, silu_on, grads)
    torch.testing.assert_close(ref["y"], y.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(ref["last"], last.detach(), rtol=0, atol=0)
    for name, v in zip(leaves, got):
        torch.testing.assert_close(ref["d" + name], v, rtol=1e-12, atol=1e-12, msg=name)


# ------------------------------------------------------------------ refusals of the C entries ----


def _p():
    buf = (ctypes.c_char * 4096)()
    return buf, (ctypes.addressof(buf) + 15) // 16 * 16


def ssm_args(p, **kw):
    a = capi.SsmArgs(batch=2, channels=4, groups=2, states=3, T=8, dtype=capi.FMS_F32, tokens=p, delta=p, B=p, C=p, A=p)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def conv_args(p, **kw):
    a = capi.ConvArgs(batch=2, channels=4, taps=4, T=8, dtype=capi.FMS_F32, tokens=p, weight=p)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(dtype=9), capi.FMS_ERR_BAD_DTYPE), (dict(batch=-1), capi.FMS_ERR_BAD_SHAPE), (dict(T=-1), capi.FMS_ERR_BAD_SHAPE),
    (dict(groups=3), capi.FMS_ERR_BAD_SHAPE), (dict(groups=0), capi.FMS_ERR_BAD_SHAPE), (dict(states=0), capi.FMS_ERR_BAD_SHAPE),
    (dict(states=257), capi.FMS_ERR_TOO_LARGE), (dict(T=2 ** 31), capi.FMS_ERR_TOO_LARGE),
    (dict(batch=2 ** 40, channels=2 ** 20), capi.FMS_ERR_BAD_SHAPE), (dict(A=None), capi.FMS_ERR_NULL_POINTER),
    (dict(tokens=None), capi.FMS_ERR_NULL_POINTER), (dict(B=None), capi.FMS_ERR_NULL_POINTER)])
def test_scan_entry_refuses(change, status):
    keep, p = _p()
    a = ssm_args(p, **change)
    assert capi.call("fms_ssm_forward", a, p, None, None, None, 0, None, check=False) == status
    if change.get("T") is None or change["T"] < 0:
        assert capi.call("fms_ssm_backward", a, p, p, None, p, p, None, p, p, p, None, None, None, p, 1 << 30, None,
                         check=False) == status


def test_scan_entry_refuses_pointers_and_scratch():
    keep, p = _p()
    a = ssm_args(p)
    fwd = lambda a, out: capi.call("fms_ssm_forward", a, out, None, None, None, 0, None, check=False)
    assert fwd(None, p) == capi.FMS_ERR_NULL_POINTER
    assert fwd(a, None) == capi.FMS_ERR_NULL_POINTER
    assert fwd(ssm_args(p, delta=p + 2), p) == capi.FMS_ERR_MISALIGNED
    assert fwd(ssm_args(p, A=p + 2), p) == capi.FMS_ERR_MISALIGNED
    assert fwd(ssm_args(p, lengths=p + 4), p) == capi.FMS_ERR_MISALIGNED
    assert fwd(ssm_args(None, batch=0, A=None), None) == capi.FMS_OK
    need = capi.lib().fms_ssm_backward_workspace_bytes(a)
    assert need > 0
    bwd = lambda ck, dz, ws, n, **kw: capi.call("fms_ssm_backward", ssm_args(p, **kw), ck, p, None, p, p, dz, p, p, p, None, None,
                                                None, ws, n, None, check=False)
    assert bwd(p, None, p, need - 1) == capi.FMS_ERR_WORKSPACE
    assert bwd(p, None, None, need) == capi.FMS_ERR_WORKSPACE
    assert bwd(None, None, p, need) == capi.FMS_ERR_NULL_POINTER
    assert bwd(p, None, p, need, z=p) == capi.FMS_ERR_NULL_POINTER     # z without a place for its gradient
    assert capi.lib().fms_ssm_checkpoint_bytes(ssm_args(p, T=65)) == 2 * 4 * 3 * 2 * 4
    assert capi.lib().fms_ssm_checkpoint_bytes(ssm_args(p, dtype=7)) == 0


def test_step_entries_refuse():
    keep, p = _p()
    step = lambda pool, slots=None, state=p, **kw: capi.call("fms_ssm_step", ssm_args(p, **{"T": 1, **kw}), state, pool, slots, p,
                                                             None, check=False)
    assert step(2, T=2) == capi.FMS_ERR_BAD_SHAPE
    assert step(1) == capi.FMS_ERR_BAD_SHAPE              # two rows, one state, no slots
    assert step(-1, slots=p) == capi.FMS_ERR_BAD_SHAPE
    assert step(2, state=None) == capi.FMS_ERR_NULL_POINTER
    assert step(2, state=p + 2) == capi.FMS_ERR_MISALIGNED
    assert step(2, slots=p + 4) == capi.FMS_ERR_MISALIGNED
    conv = lambda pool, slots=None, state=p, **kw: capi.call("fms_conv_step", conv_args(p, **{"T": 1, **kw}), state, pool, slots, p,
                                                             None, check=False)
    assert conv(2, T=2) == capi.FMS_ERR_BAD_SHAPE
    assert conv(1) == capi.FMS_ERR_BAD_SHAPE
    assert conv(2, state=None) == capi.FMS_ERR_NULL_POINTER


@pytest.mark.parametrize("change,status", [
    (dict(dtype=9), capi.FMS_ERR_BAD_DTYPE), (dict(channels=-1), capi.FMS_ERR_BAD_SHAPE), (dict(taps=1), capi.FMS_ERR_BAD_SHAPE),
    (dict(taps=9), capi.FMS_ERR_BAD_SHAPE), (dict(T=2 ** 31), capi.FMS_ERR_TOO_LARGE), (dict(weight=None), capi.FMS_ERR_NULL_POINTER),
    (dict(tokens=None), capi.FMS_ERR_NULL_POINTER), (dict(batch=2 ** 56), capi.FMS_ERR_BAD_SHAPE)])
def test_filter_entry_refuses(change, status):
    keep, p = _p()
    assert capi.call("fms_conv_forward", conv_args(p, **change), p, None, None, check=False) == status
    assert capi.call("fms_conv_backward", conv_args(p, **change), p, None, p, p, None, None, p, 1 << 30, None, check=False) == status
    need = capi.lib().fms_conv_backward_workspace_bytes(conv_args(p))
    assert capi.call("fms_conv_backward", conv_args(p), p, None, p, p, None, None, p, need - 1, None,
                     check=False) == capi.FMS_ERR_WORKSPACE


def test_ops_refuse_cpu_tensors_and_bad_arguments():
    import fm_b200
    x, A = torch.zeros(1, 2, 4), -torch.ones(2, 3)
    bc = torch.zeros(1, 3, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        fm_b200.ssm_scan(x, x, A, bc, bc)
    with pytest.raises(RuntimeError, match="CUDA"):
        fm_b200.short_conv(x, torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        fm_b200.short_conv_step(x[..., 0], torch.zeros(1, 2, 3), torch.zeros(2, 4))
    with pytest.raises(ValueError, match="activation"):
        fm_b200.short_conv(x, torch.zeros(2, 4), activation="relu")
    with pytest.raises(RuntimeError, match="no gradient"):
        fm_b200.ssm_step(x[..., 0].requires_grad_(True), x[..., 0], torch.zeros(1, 2, 3), A, bc[..., 0], bc[..., 0])
