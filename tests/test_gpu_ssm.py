"""The state-space scan, its token step and the short causal filter against their formulas in 64 bits.

Tolerances.  A stored value is off by half a step of its type, ``eps / 2`` relative.  The 32-bit
evaluation in front of it is a sum of products; each product's relative error is at most the number of
roundings on its path times 2^-24, so the sum is off by that count times the sum of the absolute values
(``magnitude=True`` of the reference).  A path runs through at most T decays (backward: twice).  One
decay exp(dt A) takes its argument with 20 roundings: A log2(e) and the product one each, and the time
step log(1 + exp(v)), |v| <= 8 here, 18: its exponential |v| from the argument and 4 of its own, the
quotient 3, the series 3.  The exponential turns them into 20 |dt A| relative, adds 2^-22, 4 roundings,
and the multiplication one: 20 |dt A| + 5 per position, and 3 for the position's own products.  Sums over states, channels, positions and sequences add one rounding a term.  The gate and the
time step add 64 (|z| <= 6: argument 2 |z| + 1, exponential 4, division 4; the same for softplus).
"""
import numpy as np
import pytest
import torch

import fm_b200
from tests import ssm_ref as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def scan_case(dtype, Bn, D, T, N, G=1, z=True, D_=True, bias=True, h0=False, lengths=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    n = lambda *s: torch.randn(*s, generator=g)
    i = dict(x=n(Bn, D, T).to(dt), delta=(0.5 * n(Bn, D, T)).to(dt),
             A=-(0.05 + torch.rand(D, N, generator=g) * 3), B=n(Bn, G, N, T).to(dt), C=n(Bn, G, N, T).to(dt),
             D=n(D) if D_ else None, z=n(Bn, D, T).to(dt) if z else None, delta_bias=(n(D) - 2) if bias else None,
             h0=n(Bn, D, N) if h0 else None, lengths=None if lengths is None else torch.tensor(lengths))
    grads = (n(Bn, D, T).to(dt), n(Bn, D, N) if h0 else None)
    return i, grads


def on_gpu(i):
    return {k: None if v is None else v.cuda() for k, v in i.items()}


def leaves_of(i):
    return {k: v.requires_grad_(True) for k, v in on_gpu(i).items() if v is not None and v.is_floating_point()}


def call_scan(c, softplus=True, return_state=False):
    B, C = c["B"], c["C"]
    if B.dim() == 4 and B.shape[1] == 1:
        B, C = B[:, 0], C[:, 0]
    return fm_b200.ssm_scan(c["x"], c["delta"], c["A"], B, C, D=c.get("D"), z=c.get("z"), delta_bias=c.get("delta_bias"),
                            initial_state=c.get("h0"), delta_softplus=softplus, lengths=c.get("lengths"), return_state=return_state)


def close(got, ref, mag, count, name):
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2
    arith = count * R.U * mag
    tol = arith + half * (ref.abs() + arith) + 1e-37
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25                      # half a step of its subnormals
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / tol).nan_to_num(9e9).max()):.3g} of the tolerance"


def scan_count(i, softplus, back=False):
    Bn, D, T = i["x"].shape
    N = i["A"].shape[1]
    raw = i["delta"].double() + (i["delta_bias"].double()[:, None] if i.get("delta_bias") is not None else 0)
    dt = R.softplus(raw) if softplus else raw
    worst = float(dt.nan_to_num(0).abs().max() * i["A"].abs().max()) if T else 0.0
    count = T * (20 * worst + 5) + 3 + N + 64
    return count * 2 + D + Bn * T if back else count


def check_scan(i, grads, softplus=True):
    want = grads[1] is not None
    c = {**on_gpu(i), **leaves_of(i)}
    outs = call_scan(c, softplus, want)
    outs = outs if want else (outs,)
    ref, mag = R.ssm(i, softplus, grads), R.ssm(i, softplus, grads, magnitude=True)
    k = scan_count(i, softplus)
    close(outs[0], ref["y"], mag["y"], k, "y")
    if want:
        close(outs[1], ref["last"], mag["last"], k, "last")
    names = [n for n in ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0") if i.get(n) is not None]
    got = torch.autograd.grad(outs, [c[n] for n in names], [v.cuda() for v in grads if v is not None])
    k = scan_count(i, softplus, back=True)
    for n, v in zip(names, got):
        assert v.dtype == i[n].dtype and v.shape == i[n].shape
        close(v, ref["d" + n], mag["d" + n], k, "d" + n)


# dtype, B, D, T, N, G, z, D, bias, h0, lengths
SCANS = [
    ("f32", 1, 1, 1, 1, 1, False, False, False, False, None),
    ("f32", 1, 4, 7, 3, 1, True, True, True, True, None),
    ("f32", 2, 5, 8, 4, 1, False, True, False, False, None),
    ("bf16", 2, 9, 63, 16, 1, True, True, True, False, None),
    ("f16", 1, 33, 64, 16, 1, True, False, True, True, None),
    ("f32", 2, 8, 65, 16, 2, True, True, True, True, None),
    ("bf16", 1, 6, 129, 17, 3, False, True, True, True, None),
    ("f16", 3, 4, 72, 16, 1, True, True, True, True, [72, 0, 5]),
    ("f32", 3, 12, 200, 20, 4, True, True, True, True, [64, 199, 65]),
    ("bf16", 2, 70, 136, 16, 1, True, True, True, False, [136, 71]),
    ("f32", 1, 131, 40, 16, 1, False, False, True, False, None),
    ("f32", 1, 3, 70, 64, 1, True, True, True, True, None),
    ("bf16", 1, 2, 66, 130, 1, True, True, True, True, None),
    ("f16", 1, 2, 9, 256, 1, False, True, True, False, None),
    ("f32", 4, 300, 16, 16, 1, True, True, True, False, None),
]


@pytest.mark.parametrize("case", SCANS, ids=lambda c: "-".join(map(str, c[:6])))
@pytest.mark.parametrize("softplus", [True, False])
def test_scan_and_gradients_match_the_formula(case, softplus):
    i, grads = scan_case(*case, seed=len(str(case)))
    if not softplus:                                # time steps as they are given: small and positive
        i["delta"] = i["delta"].abs() / 4
        i["delta_bias"] = None
    check_scan(i, grads, softplus)


# few rows and a long time: the time is cut into pieces that are scanned side by side
LONG = [("f32", 1, 2, 1100, 16, 1, True, True, True, True, None), ("bf16", 2, 5, 1001, 20, 1, False, True, True, True, [1001, 130]),
        ("f16", 1, 40, 2048, 16, 2, True, True, True, False, None), ("f32", 3, 4, 1500, 3, 1, True, False, True, True, [64, 0, 1499])]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(map(str, c[:6])))
def test_scan_of_few_long_rows(case):
    check_scan(*scan_case(*case, seed=77))


@pytest.mark.parametrize("T", [2, 15, 16, 17, 127, 128, 130])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scan_of_every_residue(T, dtype):
    check_scan(*scan_case(dtype, 2, 3, T, 5, h0=True, seed=T))


def test_scan_gradient_against_differences():
    i, grads = scan_case("f32", 2, 6, 90, 7, h0=True, seed=4)
    c = {**on_gpu(i), **leaves_of(i)}
    outs = call_scan(c, True, True)
    names = ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0")
    got = torch.autograd.grad(outs, [c[n] for n in names], [v.cuda() for v in grads])
    j = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in i.items()}
    f = lambda w: sum((a.double() * b).sum() for a, b in zip(grads, (lambda r: (r["y"], r["last"]))(R.ssm(w, True))))
    g = torch.Generator().manual_seed(1)
    for n, v in zip(names, got):
        d, e = torch.randn(i[n].shape, generator=g, dtype=torch.float64), 1e-6
        num = (f({**j, n: j[n] + e * d}) - f({**j, n: j[n] - e * d})) / (2 * e)
        # the differences are exact to 1e-7 of the terms; the gradient to fp32 roundings of them
        terms = float((v.double().cpu().abs() * d.abs()).sum())
        assert abs(float((v.double().cpu() * d).sum() - num)) <= 1e-4 * terms, n


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -3e38])
def test_scan_ignores_what_stands_behind_a_sequence(junk):
    i, grads = scan_case("f32", 3, 5, 100, 6, h0=True, lengths=[0, 33, 100], seed=8)
    k = {**i}
    for n in ("x", "delta", "z", "B", "C"):
        v = k[n] = k[n].clone()
        v[0], v[1, ..., 33:] = junk, junk
    dy = grads[0].clone()
    dy[0], dy[1, :, 33:] = junk, junk
    results = []
    for a, up in ((i, grads[0]), (k, dy)):
        c = {**on_gpu(a), **leaves_of(a)}
        outs = call_scan(c, True, True)
        names = ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0")
        results.append([*outs, *torch.autograd.grad(outs, [c[n] for n in names], [up.cuda(), grads[1].cuda()])])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    y, last, dx, dd, _, dB, dC, _, dz, _, dh0 = results[0]
    assert torch.equal(last[0].cpu(), i["h0"][0]) and torch.equal(dh0[0].cpu(), grads[1][0])
    for v in (y, dx, dd, dz):
        assert not v[0].any() and not v[1, :, 33:].any() and v[1, :, :33].any()
    assert not dB[0].any() and not dC[1, ..., 33:].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("T, at", [(60, 29), (700, 64), (700, 351), (701, 351)])
def test_a_bad_position_reaches_no_earlier_output_and_no_later_gradient(T, at, bad):
    i, grads = scan_case("bf16", 2, 9, T, 16, seed=31)
    y = call_scan(on_gpu(i))
    for n in ("x", "delta", "B", "C", "z"):
        k = {**i, n: i[n].clone()}
        k[n][0, ..., at] = bad
        z = call_scan(on_gpu(k))
        assert torch.equal(z[1], y[1]) and torch.equal(z[0, :, :at], y[0, :, :at])
        assert n == "delta" or not z[0, :, at].isfinite().any()     # an infinite time step forgets all
    dy = grads[0].clone()
    dy[0, :, at] = bad
    res = []
    for up in (grads[0], dy):
        c = {**on_gpu(i), **leaves_of(i)}
        res.append(torch.autograd.grad(call_scan(c), [c[n] for n in ("x", "delta", "z", "B", "C")], up.cuda()))
    for a, b in zip(*res):
        assert torch.equal(a[1], b[1]) and torch.equal(a[0, ..., at + 1:], b[0, ..., at + 1:])


def test_scan_lengths_are_clamped():
    i, _ = scan_case("f32", 3, 2, 20, 3, lengths=[-5, 10 ** 12, 7])
    j = {**i, "lengths": torch.tensor([0, 20, 7])}
    assert torch.equal(call_scan(on_gpu(i)), call_scan(on_gpu(j)))
    k = {**on_gpu(i), "lengths": torch.tensor([0, 20, 7], dtype=torch.int32, device="cuda")}
    assert torch.equal(call_scan(on_gpu(i)), call_scan(k))


def test_scan_takes_strided_broadcast_and_transposed_inputs():
    i, grads = scan_case("bf16", 2, 8, 48, 16, h0=True, seed=21)
    c = on_gpu(i)
    want = call_scan(c, True, True)
    xz = torch.stack([c["x"], c["z"]], 1).flatten(1, 2)                       # the two halves of one projection
    x, z = xz.chunk(2, dim=1)
    assert not x.is_contiguous()
    delta = c["delta"].transpose(1, 2).contiguous().transpose(1, 2)           # time not the contiguous axis
    wide = torch.zeros(2, 40, 64, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:19, 5:53], wide[:, 19:35, 5:53] = c["B"][:, 0], c["C"][:, 0]    # rows off the 16-byte grid
    k = {**c, "x": x, "z": z, "delta": delta, "B": wide[:, None, 3:19, 5:53], "C": wide[:, None, 19:35, 5:53]}
    got = call_scan(k, True, True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # one sequence's B for the whole batch: the gradient is summed over the batch
    one = c["B"][:1, 0].clone().requires_grad_(True)
    y = fm_b200.ssm_scan(c["x"], c["delta"], c["A"], one.expand(2, -1, -1), c["C"][:, 0], delta_softplus=True)
    (d_one,) = torch.autograd.grad(y, one, grads[0].cuda())
    both = c["B"][:1, 0].repeat(2, 1, 1).requires_grad_(True)
    y2 = fm_b200.ssm_scan(c["x"], c["delta"], c["A"], both, c["C"][:, 0], delta_softplus=True)
    (d_both,) = torch.autograd.grad(y2, both, grads[0].cuda())
    assert torch.equal(y, y2)
    torch.testing.assert_close(d_one, d_both.sum(0, keepdim=True), rtol=2 ** -7, atol=1e-3)


def test_scan_gradient_of_an_expanded_upstream():
    i, _ = scan_case("f32", 2, 4, 30, 4, seed=5)
    c = {**on_gpu(i), **leaves_of(i)}
    a = torch.autograd.grad(call_scan(c).sum(), c["x"])[0]
    b = torch.autograd.grad(call_scan(c), c["x"], torch.ones(2, 4, 30, device="cuda"))[0]
    assert torch.equal(a, b)


def test_scan_state_alone_and_output_alone():
    i, grads = scan_case("f32", 2, 4, 30, 4, h0=True, seed=6)
    for pick, up in ((1, grads[1]), (0, grads[0])):
        c = {**on_gpu(i), **leaves_of(i)}
        out = call_scan(c, True, True)[pick]
        got = torch.autograd.grad(out, c["x"], up.cuda())[0]
        zero = (torch.zeros_like(grads[0]), grads[1]) if pick else (grads[0], torch.zeros_like(grads[1]))
        ref, mag = R.ssm(i, True, zero), R.ssm(i, True, zero, magnitude=True)
        close(got, ref["dx"], mag["dx"], scan_count(i, True, back=True), "dx")


def test_empty_scans():
    i, _ = scan_case("f32", 2, 3, 0, 4, h0=True)
    y, last = call_scan(on_gpu(i), True, True)
    assert y.shape == (2, 3, 0) and torch.equal(last.cpu(), i["h0"])
    c = {**on_gpu(i), **leaves_of(i)}
    y, last = call_scan(c, True, True)
    d, dA = torch.autograd.grad(last.sum() + y.sum(), [c["h0"], c["A"]])
    assert torch.equal(d, torch.ones_like(d)) and not dA.any()
    i, _ = scan_case("f32", 0, 3, 5, 4)
    c = {**on_gpu(i), **leaves_of(i)}
    y = call_scan(c)
    assert y.shape == (0, 3, 5) and not torch.autograd.grad(y.sum(), c["A"])[0].any()


def test_scan_gives_equal_bits_twice_and_on_another_stream():
    i, grads = scan_case("bf16", 3, 200, 700, 16, h0=True, seed=31)
    def once():
        c = {**on_gpu(i), **leaves_of(i)}
        outs = call_scan(c, True, True)
        return [*outs, *torch.autograd.grad(outs, [c[n] for n in ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0")],
                                            [g.cuda() for g in grads])]
    first, second = once(), once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    other = []
    for s in streams:                                # two at once
        with torch.cuda.stream(s):
            other.append(once())
    torch.cuda.synchronize()
    for a, b, c, d in zip(first, second, *other):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)


def test_scan_step_and_filter_replay_from_a_graph():
    i, grads = scan_case("bf16", 2, 32, 100, 16, h0=True, seed=12)
    c = {**on_gpu(i), **leaves_of(i)}
    w = torch.randn(32, 4, device="cuda", requires_grad=True)
    up = [g.cuda() for g in grads]
    state = torch.randn(2, 32, 16, device="cuda")
    names = [c["x"], c["A"], c["B"], w]
    tok = [c[k].detach()[..., 0].clone() for k in ("x", "delta")]
    bc = [c[k].detach()[:, 0, :, 0].clone() for k in ("B", "C")]

    def work():
        f = fm_b200.short_conv(c["x"], w, activation="silu")
        y, last = call_scan({**c, "x": f}, True, True)
        g = torch.autograd.grad((y, last), names, up)
        with torch.no_grad():
            t = fm_b200.ssm_step(*tok, state, c["A"], *bc, delta_softplus=True)
        return [y, last, *g, t]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            work()
    torch.cuda.current_stream().wait_stream(s)
    start = torch.randn(2, 32, 16, device="cuda")
    state.copy_(start)
    want = [v.detach().clone() for v in work()]
    after = state.clone()
    graphs, outs = [], []
    for _ in range(2):                               # two graphs of the same work, side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work())
        graphs.append(g)
    for g, o in zip(graphs, outs):
        state.copy_(start)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(o, want):
            assert torch.equal(a, b)
        assert torch.equal(state, after)


def test_scan_offsets_pass_32_bits():
    D, T = 34, 1 << 26                               # 2.3e9 positions in one tensor
    x = torch.ones(1, D, T, device="cuda", dtype=torch.bfloat16)
    delta = torch.full((1, 1, 1), 0.25, device="cuda", dtype=torch.bfloat16).expand(1, D, T).contiguous()
    A = -torch.ones(D, 1, device="cuda")
    bc = torch.ones(1, 1, T, device="cuda", dtype=torch.bfloat16)
    x[0, -1, -100:] = torch.arange(100, device="cuda")
    y, last = fm_b200.ssm_scan(x, delta, A, bc, bc, return_state=True)
    # far from the start every channel stands at its fixed point 0.25 / (1 - exp(-0.25))
    z, last1 = fm_b200.ssm_scan(x[:, -1:, -4096:], delta[:, -1:, -4096:], A[:1], bc[..., -4096:], bc[..., -4096:], return_state=True)
    assert torch.equal(y[0, -1, -1024:], z[0, 0, -1024:])
    torch.testing.assert_close(last[0, -1], last1[0, 0], rtol=1e-6, atol=0)
    f = fm_b200.short_conv(x, torch.ones(D, 4, device="cuda"))
    assert torch.equal(f[0, -1, -3:].float(), (4 * torch.tensor([97., 98., 99.], device="cuda") - 6).bfloat16().float())
    assert torch.equal(f[0, -1, :4].float().cpu(), torch.tensor([1., 2., 3., 4.]))


def test_no_gradient_needed_keeps_no_states_and_second_order_is_refused():
    i, _ = scan_case("f32", 1, 2, 10, 2)
    assert not call_scan(on_gpu(i)).requires_grad
    c = {**on_gpu(i), **leaves_of(i)}
    (g,) = torch.autograd.grad(call_scan(c).square().sum(), c["x"], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---------------------------------------------------------------------------------- one token ----


@pytest.mark.parametrize("dtype,Bn,D,N,G,z", [("f32", 1, 1, 1, 1, False), ("bf16", 3, 130, 16, 1, True), ("f16", 2, 6, 5, 3, True),
                                              ("f32", 4, 12, 64, 2, False), ("bf16", 1, 3, 256, 1, True), ("f32", 2, 33, 8, 1, True)])
def test_step_matches_the_formula(dtype, Bn, D, N, G, z):
    i, _ = scan_case(dtype, Bn, D, 1, N, G, z=z, h0=True, seed=N)
    ref, mag = R.ssm(i, True), R.ssm(i, True, magnitude=True)
    c = on_gpu(i)
    pool = Bn + 2
    state = torch.randn(pool, D, N, device="cuda")
    slots = torch.randperm(pool, device="cuda")[:Bn]
    state[slots] = c["h0"]
    before = state.clone()
    bc = lambda v: v[..., 0] if G > 1 else v[:, 0, :, 0]
    y = fm_b200.ssm_step(c["x"][..., 0], c["delta"][..., 0], state, c["A"], bc(c["B"]), bc(c["C"]), D=c["D"],
                         z=None if c["z"] is None else c["z"][..., 0], delta_bias=c["delta_bias"], delta_softplus=True, slots=slots)
    k = scan_count(i, True)
    close(y, ref["y"][..., 0], mag["y"][..., 0], k, "y")
    close(state[slots], ref["last"], mag["last"], k, "state")
    rest = [r for r in range(pool) if r not in slots.tolist()]
    assert torch.equal(state[rest], before[rest])


def test_steps_skip_padding_far_and_repeated_slots():
    D, N, K = 20, 16, 4
    g = torch.Generator(device="cuda").manual_seed(2)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    slots = torch.tensor([2, -1, 4, 2, 5, 2 ** 40, 0, -2 ** 60, 4], device="cuda")
    own = [0, 2, 6]                                  # the rows that have a state of their own (5 is outside a pool of 5)
    x, d, B, C, A = n(9, D), n(9, D), n(9, N), n(9, N), -torch.rand(D, N, device="cuda")
    first = n(5, D, N)
    state = first.clone()
    y = fm_b200.ssm_step(x, d, state, A, B, C, delta_softplus=True, slots=slots)
    want = first.clone()
    alone = first[slots[own]].contiguous()
    ya = fm_b200.ssm_step(x[own], d[own], alone, A, B[own], C[own], delta_softplus=True)
    want[slots[own]] = alone
    assert torch.equal(state, want) and torch.equal(y[own], ya)
    rest = [r for r in range(9) if r not in own]
    assert not y[rest].any()
    w = n(D, K)
    first = n(5, D, K - 1)
    state = first.clone()
    y = fm_b200.short_conv_step(x, state, w, slots=slots.clone())
    want = first.clone()
    alone = first[slots[own]].contiguous()
    ya = fm_b200.short_conv_step(x[own], alone, w)
    want[slots[own]] = alone
    assert torch.equal(state, want) and torch.equal(y[own], ya) and not y[rest].any()
    assert torch.equal(alone, torch.cat([first[slots[own]][..., 1:], x[own][..., None]], -1))


def test_step_of_a_wide_batch_finds_repeats_beyond_one_block():
    Bn, D, N = 1000, 3, 4
    slots = torch.arange(Bn, device="cuda") % 700    # the last 300 rows repeat
    g = torch.Generator(device="cuda").manual_seed(3)
    x, d, B = (torch.randn(Bn, k, generator=g, device="cuda") for k in (D, D, N))
    state = torch.randn(700, D, N, generator=g, device="cuda")
    once = state.clone()
    A = -torch.ones(D, N, device="cuda")
    y = fm_b200.ssm_step(x, d, state, A, B, B, delta_softplus=True, slots=slots)
    y1 = fm_b200.ssm_step(x[:700], d[:700], once, A, B[:700], B[:700], delta_softplus=True)
    assert torch.equal(state, once) and torch.equal(y[:700], y1) and not y[700:].any()


def test_step_reaches_states_behind_32_bit_offsets():
    D, N, pool = 2048, 16, 65540                     # 2.1e9 floats
    state = torch.zeros(pool, D, N, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, d, B, C, A = n(2, D), n(2, D), n(2, N), n(2, N), -torch.rand(D, N, generator=g, device="cuda")
    small = n(2, D, N)
    slots = torch.tensor([pool - 1, 65536], device="cuda")
    state[slots] = small
    y = fm_b200.ssm_step(x, d, state, A, B, C, delta_softplus=True, slots=slots)
    y1 = fm_b200.ssm_step(x, d, small, A, B, C, delta_softplus=True)
    assert torch.equal(y, y1) and torch.equal(state[slots], small) and not state[:65536].any()


# ------------------------------------------------------------------------------------- filter ----


def conv_case(dtype, Bn, D, T, K, bias, x0, lengths, seed):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    n = lambda *s: torch.randn(*s, generator=g)
    i = dict(x=n(Bn, D, T).to(dt), w=n(D, K), b=n(D) if bias else None, x0=n(Bn, D, K - 1).to(dt) if x0 else None,
             lengths=None if lengths is None else torch.tensor(lengths))
    return i, (n(Bn, D, T).to(dt), n(Bn, D, K - 1).to(dt) if x0 else None)


CONVS = [("f32", 1, 1, 1, 4, False, False, None), ("f32", 2, 3, 2, 4, True, True, None), ("bf16", 2, 5, 7, 8, True, True, None),
         ("f16", 1, 4, 8, 2, True, False, None), ("f32", 3, 7, 9, 3, True, True, [9, 0, 1]), ("bf16", 2, 6, 64, 5, False, True, [3, 64]),
         ("f32", 1, 5, 255, 4, True, True, None), ("bf16", 3, 3, 256, 4, True, True, None), ("f16", 2, 3, 257, 6, True, True, None),
         ("bf16", 1, 3, 1023, 4, True, False, None), ("f32", 2, 2, 1024, 7, True, True, [1024, 1022]),
         ("bf16", 2, 3, 1032, 4, True, True, [1032, 1026]), ("f32", 2, 3, 2500, 8, True, True, [2049, 1024]),
         ("f16", 1, 260, 40, 4, True, True, None)]


@pytest.mark.parametrize("case", CONVS, ids=lambda c: "-".join(map(str, c[:5])))
@pytest.mark.parametrize("act", [None, "silu"])
def test_filter_and_gradients_match_the_formula(case, act):
    i, grads = conv_case(*case, seed=case[3] + case[4])
    c = {**on_gpu(i), **leaves_of(i)}
    want = grads[1] is not None
    outs = fm_b200.short_conv(c["x"], c["w"], c.get("b"), initial_state=c.get("x0"), activation=act, lengths=c["lengths"],
                              return_state=want)
    outs = outs if want else (outs,)
    ref, mag = R.conv(i, act == "silu", grads), R.conv(i, act == "silu", grads, magnitude=True)
    Bn, D, T = i["x"].shape
    K = i["w"].shape[1]
    close(outs[0], ref["y"], mag["y"], K + 64, "y")
    if want:
        assert torch.equal(outs[1].double().cpu(), ref["last"])
    names = [n for n in ("x", "w", "b", "x0") if i.get(n) is not None]
    got = torch.autograd.grad(outs, [c[n] for n in names], [v.cuda() for v in grads if v is not None])
    for n, v in zip(names, got):
        assert v.dtype == i[n].dtype
        close(v, ref["d" + n], mag["d" + n], 2 * K + 128 + (Bn * T if n in "wb" else 0), "d" + n)


@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_filter_ignores_what_stands_behind_a_sequence_and_reads_no_further_than_its_taps(junk):
    i, grads = conv_case("f32", 2, 3, 300, 4, True, True, [300, 130], 5)
    k = {**i, "x": i["x"].clone()}
    k["x"][1, :, 130:] = junk
    dy = grads[0].clone()
    dy[1, :, 130:] = junk
    res = []
    for a, up in ((i, grads[0]), (k, dy)):
        c = {**on_gpu(a), **leaves_of(a)}
        outs = fm_b200.short_conv(c["x"], c["w"], c["b"], c["x0"], "silu", c["lengths"], True)
        res.append([*outs, *torch.autograd.grad(outs, [c[n] for n in ("x", "w", "b", "x0")], [up.cuda(), grads[1].cuda()])])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    assert not res[0][0][1, :, 130:].any() and not res[0][2][1, :, 130:].any()
    x = torch.zeros(1, 1, 64, device="cuda")
    x[0, 0, 20] = junk
    y = fm_b200.short_conv(x, torch.ones(1, 4, device="cuda"))
    assert y[0, 0, :20].isfinite().all() and y[0, 0, 24:].isfinite().all() and not y[0, 0, 20:24].isfinite().any()


def test_filter_takes_strided_and_offset_rows():
    g = torch.Generator(device="cuda").manual_seed(7)
    wide = torch.randn(2, 10, 700, generator=g, device="cuda").bfloat16()
    x, w = wide[:, 2:7, 3:600], torch.randn(5, 4, generator=g, device="cuda")
    assert torch.equal(fm_b200.short_conv(x, w), fm_b200.short_conv(x.contiguous(), w))
    t = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(fm_b200.short_conv(t, w), fm_b200.short_conv(x.contiguous(), w))


def test_filter_of_no_positions_passes_its_state_on():
    x = torch.zeros(2, 3, 0, device="cuda", requires_grad=True)
    w = torch.randn(3, 4, device="cuda", requires_grad=True)
    x0 = torch.randn(2, 3, 3, device="cuda", requires_grad=True)
    y, last = fm_b200.short_conv(x, w, initial_state=x0, return_state=True)
    assert y.shape == (2, 3, 0) and torch.equal(last, x0)
    up = torch.randn(2, 3, 3, device="cuda")
    dw, d0 = torch.autograd.grad((y, last), (w, x0), (torch.zeros_like(y), up))
    assert torch.equal(d0, up) and not dw.any()


def test_more_sequences_than_a_grid_axis_holds():
    Bn, K = 65_600, 4
    g = torch.Generator(device="cuda").manual_seed(8)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w, up = n(Bn, 1, 5).requires_grad_(True), n(1, K).requires_grad_(True), n(Bn, 1, 5)
    y = fm_b200.short_conv(x, w)
    want = torch.nn.functional.conv1d(torch.nn.functional.pad(x.double(), (K - 1, 0)), w.double()[:, None])
    # each output is a sum of 4 products
    assert ((y.double() - want).abs() <= 8 * R.U * 64).all()
    dx, dw = torch.autograd.grad(y, (x, w), up)
    wx, ww = torch.autograd.grad(want, (x, w), up.double())
    assert ((dx - wx).abs() <= 8 * R.U * 64).all()
    assert ((dw - ww).abs() <= (5 * Bn + 8) ** 0.5 * 64 * R.U * 64 * 5).all()
    state = n(Bn, 1, K - 1)
    s2 = state.clone()
    a = fm_b200.short_conv_step(x[..., 0].detach(), state, w.detach())
    b = fm_b200.short_conv_step(x[65_500:, :, 0].detach(), s2[65_500:].contiguous(), w.detach())
    assert torch.equal(a[65_500:], b)
    h = n(Bn, 1, 8)
    h2 = h[65_500:].clone()
    A, bc = -torch.ones(1, 8, device="cuda"), n(Bn, 8)
    a = fm_b200.ssm_step(x[..., 0].detach(), x[..., 1].detach(), h, A, bc, bc, delta_softplus=True)
    b = fm_b200.ssm_step(x[65_500:, :, 0].detach(), x[65_500:, :, 1].detach(), h2, A, bc[65_500:], bc[65_500:], delta_softplus=True)
    assert torch.equal(a[65_500:], b) and torch.equal(h[65_500:], h2)
    z = fm_b200.ssm_scan(x.detach(), x.detach(), A, n(Bn, 8, 5), n(Bn, 8, 5), delta_softplus=True)
    assert z.isfinite().all()


# -------------------------------------------------------------------------------- all together ----


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_layer_prompt_then_tokens_equals_the_whole_sequence(dtype):
    """Filter, projections, scan: a padded batch of prompts, then token by token on a pool; against one pass."""
    dt, Bn, D, T, N, K, more = DT[dtype], 3, 24, 40, 16, 4, 6
    g = torch.Generator(device="cuda").manual_seed(17)
    n = lambda *s, scale=1.0: torch.randn(*s, generator=g, device="cuda") * scale
    w, b, A = n(D, K), n(D), -torch.rand(D, N, generator=g, device="cuda") * 3
    proj, D_, bias = n(D + 2 * N, D, scale=D ** -0.5).to(dt), n(D), n(D) - 2
    x, z = n(Bn, D, T + more).to(dt), n(Bn, D, T + more).to(dt)
    prompt = torch.tensor([T, 11, 29], device="cuda")

    def layer(xs, zs, x0, h0, lengths):
        f, x_last = fm_b200.short_conv(xs, w, b, initial_state=x0, activation="silu", lengths=lengths, return_state=True)
        p = proj @ f
        y, h = fm_b200.ssm_scan(f, p[:, :D], A, p[:, D:D + N], p[:, D + N:], D=D_, z=zs, delta_bias=bias, initial_state=h0,
                                delta_softplus=True, lengths=lengths, return_state=True)
        return y, x_last, h

    with torch.no_grad():
        whole, _, h_end = layer(x, z, None, None, prompt + more)
        y, x_last, h = layer(x[..., :T], z[..., :T], None, None, prompt)
        slots = torch.tensor([4, 0, 2], device="cuda")
        conv_pool, state_pool = torch.zeros(5, D, K - 1, device="cuda", dtype=dt), torch.zeros(5, D, N, device="cuda")
        conv_pool[slots], state_pool[slots] = x_last, h
        tol = dict(rtol=1e-4, atol=1e-4) if dtype == "f32" else dict(rtol=0.05, atol=0.05)
        for r in range(Bn):
            torch.testing.assert_close(y[r, :, :prompt[r]], whole[r, :, :prompt[r]], **tol)
        rows = torch.arange(Bn, device="cuda")
        for t in range(more):
            at = prompt + t
            f = fm_b200.short_conv_step(x[rows, :, at], conv_pool, w, b, activation="silu", slots=slots)
            p = f @ proj.T
            out = fm_b200.ssm_step(f, p[:, :D], state_pool, A, p[:, D:D + N], p[:, D + N:], D=D_, z=z[rows, :, at],
                                   delta_bias=bias, delta_softplus=True, slots=slots)
            torch.testing.assert_close(out, whole[rows, :, at], **tol)
        torch.testing.assert_close(state_pool[slots], h_end, **tol)
        assert not state_pool[[1, 3]].any() and not conv_pool[[1, 3]].any()


def test_refusals():
    i, _ = scan_case("f32", 2, 4, 10, 3)
    c = on_gpu(i)
    ok = dict(x=c["x"], delta=c["delta"], A=c["A"], B=c["B"][:, 0], C=c["C"][:, 0])
    run = lambda **kw: (lambda a, more: fm_b200.ssm_scan(a["x"], a["delta"], a["A"], a["B"], a["C"], **more))(
        {**ok, **{k: v for k, v in kw.items() if k in ok}}, {k: v for k, v in kw.items() if k not in ok})
    run()
    for kw, text in ((dict(delta=c["delta"].half()), "dtype"), (dict(delta=c["delta"][:, :3]), "shape"), (dict(A=c["A"][:3]), "shape"),
                     (dict(B=c["B"][:, 0, :2]), "shape"), (dict(B=c["B"].expand(2, 3, 3, 10), C=c["C"].expand(2, 3, 3, 10)), "divide"),
                     (dict(z=c["x"][:1]), "shape"), (dict(D=torch.ones(3, device="cuda")), "shape"),
                     (dict(initial_state=torch.zeros(2, 4, 2, device="cuda")), "shape"), (dict(lengths=torch.ones(3, device="cuda").long()), "lengths"),
                     (dict(lengths=torch.ones(2).long()), "lengths"), (dict(lengths=torch.ones(2, device="cuda")), "lengths"),
                     (dict(x=c["x"].double(), delta=c["delta"].double(), B=ok["B"].double(), C=ok["C"].double()), "dtype"),
                     (dict(A=torch.zeros(4, 257, device="cuda")), "states")):
        with pytest.raises(RuntimeError, match=text):
            run(**kw)
    w = torch.ones(4, 4, device="cuda")
    for call, text in ((lambda: fm_b200.short_conv(c["x"], w[:, :1]), "taps"), (lambda: fm_b200.short_conv(c["x"], w[:3]), "shape"),
                       (lambda: fm_b200.short_conv(c["x"], w, initial_state=torch.zeros(2, 4, 2, device="cuda")), "shape"),
                       (lambda: fm_b200.short_conv(c["x"][0], w), "tokens"),
                       (lambda: fm_b200.short_conv_step(c["x"][..., 0], torch.zeros(1, 4, 3, device="cuda"), w), "one state per row"),
                       (lambda: fm_b200.short_conv_step(c["x"][..., 0], torch.zeros(2, 4, 3, device="cuda").half(), w), "dtype"),
                       (lambda: fm_b200.ssm_step(c["x"][..., 0], c["x"][..., 0], torch.zeros(2, 4, 3, device="cuda").half(), c["A"],
                                                 ok["B"][..., 0], ok["C"][..., 0]), "float32"),
                       (lambda: fm_b200.ssm_step(c["x"][..., 0], c["x"][..., 0], torch.zeros(2, 3, 4, device="cuda").transpose(1, 2), c["A"],
                                                 ok["B"][..., 0], ok["C"][..., 0]), "contiguous")):
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_tensors_on_another_device_than_the_current_one():
    i, grads = scan_case("f32", 1, 4, 20, 3)
    c = {k: v.to("cuda:1").requires_grad_(v.is_floating_point()) if v is not None else None for k, v in i.items()}
    with torch.cuda.device(0):
        y = call_scan(c)
        torch.autograd.grad(y, c["x"], grads[0].to("cuda:1"))
    assert torch.equal(y.cpu(), call_scan(on_gpu(i)).cpu())
