"""What the state-space operators are measured on: cases, inputs, plain forms and exact values.

Four operators of a selective state-space layer, all along the time axis of (B, D, T) rows like the
rest of the package:

* ``ssm_scan``         h_t = exp(dt_t A) h_{t-1} + dt_t B_t x_t,  y_t = <C_t, h_t> + D x_t, times silu(z_t)
* ``ssm_step``         the same recurrence for one token, on states kept in a pool
* ``short_conv``       depthwise causal filter of K taps in front of it, y_t = act(b + sum_k w_k x_{t-K+1+k})
* ``short_conv_step``  the same filter for one token, on the last K - 1 inputs kept in a pool

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits; with ``own``
true it makes the calls a user makes.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_MOST_SCAN = 8 * 1024 * 4096 * 16   # states (B*D*T*N) of the largest listed scan
_MOST_CONV = 8 * 2048 * 4096        # positions (B*D*T) of the largest listed filter
_MOST_STEP = 256 * 2048 * 16        # states (B*D*N) of the largest listed token step


def listed():
    return [
        # one optimizer step of a small fp32 model: latency of the whole forward and backward
        dict(name="scan train f32 small", op="scan", train=True, dtype="f32", B=2, D=64, T=1024, N=16, G=1,
             z=True, lengths=False, state=False),
        # an ordinary training step of one layer
        dict(name="scan train bf16", op="scan", train=True, dtype="bf16", B=8, D=1024, T=4096, N=16, G=1,
             z=True, lengths=False, state=False),
        # fine-tuning on a padded batch: ragged lengths, a sequence that is all padding among them
        dict(name="scan train f16 padded", op="scan", train=True, dtype="f16", B=3, D=768, T=1000, N=16, G=1,
             z=True, lengths=True, state=True),
        # one long prompt, whose last state goes on to the token steps
        dict(name="scan prompt bf16 long", op="scan", train=False, dtype="bf16", B=1, D=2048, T=8192, N=16, G=1,
             z=True, lengths=False, state=True),
        # prompts of odd length: no row starts on a vector boundary
        dict(name="scan prompt f16 odd", op="scan", train=False, dtype="f16", B=3, D=768, T=16385, N=16, G=1,
             z=False, lengths=False, state=False),
        # many short prompts continued from cached states, wide states in two groups
        dict(name="scan prompt bf16 N64", op="scan", train=False, dtype="bf16", B=16, D=1024, T=333, N=64, G=2,
             z=True, lengths=True, state=True),
        # one user's next token: latency
        dict(name="step one", op="step", dtype="bf16", B=1, D=2048, N=16, G=1, z=True, pool=1),
        # a serving batch with some padding rows: every state is read and written once
        dict(name="step batch", op="step", dtype="bf16", B=256, D=2048, N=16, G=1, z=True, pool=320),
        # an ordinary training step
        dict(name="conv train bf16", op="conv", train=True, dtype="bf16", B=8, D=2048, T=4096, K=4, silu=True,
             lengths=False, state=False),
        # prompts of odd length with the filter's state carried in and out
        dict(name="conv prompt f16 odd", op="conv", train=False, dtype="f16", B=3, D=768, T=16385, K=4, silu=True,
             lengths=False, state=True),
        # one user's next token, and a serving batch
        dict(name="conv step one", op="convstep", dtype="bf16", B=1, D=2048, K=4, silu=True, pool=1),
        dict(name="conv step batch", op="convstep", dtype="bf16", B=256, D=2048, K=4, silu=True, pool=320),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "conv", "conv", "step", "convstep"])
    c = dict(op=op, dtype=rng.choice(["f32", "f16", "bf16", "bf16"]))
    if op in ("scan", "step"):
        N = rng.choice([16, 16, 16, 8, 32, 64, rng.randint(1, 64)])
        G = rng.choice([1, 1, 1, 2, 4])
    if op in ("scan", "conv"):
        B, D, T = _log(rng, 1, 16), _log(rng, 16, 2048), _log(rng, 1, 16385)
        if op == "scan":
            D = -(-D // G) * G
        per, most = (N, _MOST_SCAN) if op == "scan" else (1, _MOST_CONV)
        T = max(1, min(T, most // (B * D * per)))
        c.update(train=rng.random() < 0.6, B=B, D=D, T=T, lengths=rng.random() < 0.3, state=rng.random() < 0.5)
    else:
        B, D = _log(rng, 1, 256), _log(rng, 16, 2048)
        if op == "step":
            D = -(-D // G) * G
            B = max(1, min(B, _MOST_STEP // (D * N)))
        c.update(B=B, D=D, pool=B + rng.choice([0, 1, B // 4]))
    if op in ("scan", "step"):
        c.update(N=N, G=G, z=rng.random() < 0.7)
    else:
        c.update(K=rng.choice([2, 3, 4, 4, 5, 8]), silu=rng.random() < 0.8)
    return c


# ------------------------------------------------------------------------------------ inputs ----


def _slots(c, randint):
    """A place in the pool for every row; the last row of a larger batch is padding (-1)."""
    order = torch.argsort(randint(0, 1 << 30, (c["pool"],)))[:c["B"]]
    if c["B"] > 3:
        order[-1] = -1
    return order


def prepare(case, seed):
    c, dt = case, _DT[case["dtype"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, dtype=dt, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def randint(lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda")

    B, D = c["B"], c["D"]
    s = dict(case=c)
    if c["op"] in ("scan", "step"):
        N, G = c["N"], c["G"]
        # decay rates spread from 1 to N and time steps from 1e-3 to 1e-1, as such layers are initialised
        s["A"] = -torch.arange(1, N + 1, device="cuda").float().expand(D, N) * torch.exp(0.1 * normal(D, N, dtype=torch.float32))
        dt0 = torch.exp(uniform(D) * (math.log(1e-1) - math.log(1e-3)) + math.log(1e-3))
        s["delta_bias"] = dt0 + torch.log(-torch.expm1(-dt0))
        s["D"] = normal(D, dtype=torch.float32, scale=0.1, mean=1.0)
    if c["op"] == "scan":
        T = c["T"]
        s["x"], s["delta"] = normal(B, D, T), normal(B, D, T, scale=0.5)
        s["z"] = normal(B, D, T) if c["z"] else None
        shape = (B, G, N, T) if G > 1 else (B, N, T)
        s["B"], s["C"] = normal(*shape), normal(*shape)
        s["h0"] = normal(B, D, N, dtype=torch.float32) if c["state"] else None
        s["dy"] = normal(B, D, T) if c["train"] else None
        s["dlast"] = normal(B, D, N, dtype=torch.float32) if c["train"] and c["state"] else None
    elif c["op"] == "step":
        shape = (B, G, N) if G > 1 else (B, N)
        s["x"], s["delta"], s["B"], s["C"] = normal(B, D), normal(B, D, scale=0.5), normal(*shape), normal(*shape)
        s["z"] = normal(B, D) if c["z"] else None
        s["state"] = normal(c["pool"], D, N, dtype=torch.float32)
        s["slots"] = _slots(c, randint)
    else:
        K = c["K"]
        s["w"] = normal(D, K, dtype=torch.float32, scale=1 / math.sqrt(K))
        s["b"] = normal(D, dtype=torch.float32, scale=0.1)
        if c["op"] == "conv":
            s["x"] = normal(B, D, c["T"])
            s["x0"] = normal(B, D, K - 1) if c["state"] else None
            s["dy"] = normal(B, D, c["T"]) if c["train"] else None
            s["dlast"] = normal(B, D, K - 1) if c["train"] and c["state"] else None
        else:
            s["x"], s["state"] = normal(B, D), normal(c["pool"], D, K - 1)
            s["slots"] = _slots(c, randint)
    if c.get("lengths") is not None:
        s["lengths"] = None
        if c["lengths"]:
            s["lengths"] = randint(0, c["T"] + 1, (B,))
            s["lengths"][0] = c["T"]
            if B > 2:
                s["lengths"][B // 2] = 0
    if c.get("train"):
        names = ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0") if c["op"] == "scan" else ("x", "w", "b", "x0")
        s["leaves"] = [n for n in names if s[n] is not None]
        for n in s["leaves"]:
            s[n].requires_grad_(True)
    return s


# ------------------------------------------------------------------------- the user's calls ----


def _run_own(s):
    import fm_b200
    c = s["case"]
    act = "silu" if c.get("silu") else None
    if c["op"] == "step":
        y = fm_b200.ssm_step(s["x"], s["delta"], s["state"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                             delta_bias=s["delta_bias"], delta_softplus=True, slots=s["slots"])
        return dict(y=y, state=s["state"])
    if c["op"] == "convstep":
        y = fm_b200.short_conv_step(s["x"], s["state"], s["w"], s["b"], activation=act, slots=s["slots"])
        return dict(y=y, state=s["state"])
    if c["op"] == "scan":
        r = fm_b200.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                             delta_bias=s["delta_bias"], initial_state=s["h0"], delta_softplus=True,
                             lengths=s["lengths"], return_state=c["state"])
    else:
        r = fm_b200.short_conv(s["x"], s["w"], s["b"], initial_state=s["x0"], activation=act,
                               lengths=s["lengths"], return_state=c["state"])
    outs = r if c["state"] else (r,)
    got = dict(zip(("y", "last"), outs))
    if c["train"]:
        ups = [s["dy"], s["dlast"]][:len(outs)]
        grads = torch.autograd.grad(outs, [s[n] for n in s["leaves"]], ups)
        got = {k: v.detach() for k, v in got.items()}
        got.update({"d" + n: v for n, v in zip(s["leaves"], grads)})
    return got


# ------------------------------------------------------------------------------ plain forms ----


def _recur(a, b):
    """h_t = a_t h_{t-1} + b_t along the last axis: log2(T) doublings of the span that is summed up."""
    k = 1
    while k < a.shape[-1]:
        b = torch.cat([b[..., :k], b[..., k:] + a[..., k:] * b[..., :-k]], -1)
        a = torch.cat([a[..., :k], a[..., k:] * a[..., :-k]], -1)
        k *= 2
    return b


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _silu(v):
    return v / (1 + torch.exp(-v))


def _dsilu(v):
    p = 1 / (1 + torch.exp(-v))
    return p * (1 + v * (1 - p))


def _inside(s, T):
    """(B, 1, T) truth: the position belongs to its sequence."""
    at = torch.arange(T, device="cuda")
    n = s["lengths"]
    return (at < T).view(1, 1, T) if n is None else at.view(1, 1, T) < n.view(-1, 1, 1)


def _grouped(v, G):
    """(B, N, T) or (B, G, N, T), in 32 bits, as (B, G, 1, N, T)."""
    return (v.float() if v.dim() == 4 else v.float()[:, None])[:, :, None]


def _plain_scan(s):
    c = s["case"]
    B, D, T, N, G, dt = c["B"], c["D"], c["T"], c["N"], c["G"], s["x"].dtype
    M = D // G
    keep = _inside(s, T)
    x = torch.where(keep, s["x"].float(), 0.0)
    raw = s["delta"].float() + s["delta_bias"][:, None]
    d = torch.where(keep, _softplus(raw), 0.0)
    Bt, Ct = (torch.where(keep[:, :, None, None], _grouped(s[n], G), 0.0) for n in ("B", "C"))
    five = (B, G, M, 1, T)
    A = s["A"].view(1, G, M, N, 1)
    h0 = torch.zeros(B, D, N, device="cuda") if s["h0"] is None else s["h0"]
    a = torch.exp(d.view(five) * A)
    b = (d * x).view(five) * Bt
    b[..., 0] += a[..., 0] * h0.view(B, G, M, N)
    h = _recur(a, b)
    y = (Ct * h).sum(3).view(B, D, T) + s["D"][:, None] * x
    out = y
    if s["z"] is not None:
        z = torch.where(keep, s["z"].float(), 0.0)
        out = y * _silu(z)
    got = dict(y=torch.where(keep, out, 0.0).to(dt))
    if c["state"]:
        got["last"] = h[..., -1].reshape(B, D, N).clone()
    if not c["train"]:
        return got
    up = torch.where(keep, s["dy"].float(), 0.0)
    dy = up
    if s["z"] is not None:
        dy = up * _silu(z)
        got["dz"] = (up * y * _dsilu(z)).to(dt)
    # adjoint of the states, from the last to the first: g_t = C_t dy_t + a_{t+1} g_{t+1}
    back = torch.cat([a[..., 1:], torch.zeros_like(a[..., :1])], -1).flip(-1)
    seed = Ct * dy.view(five)
    if c["state"]:
        seed[..., -1] += s["dlast"].view(B, G, M, N)
    g = _recur(back, seed.flip(-1)).flip(-1)
    before = torch.cat([h0.view(B, G, M, N, 1), h[..., :-1]], -1)
    q = g * a * before                                   # dL/d(dt A) of every position
    gB = (g * Bt).sum(3).view(B, D, T)
    got["dx"] = torch.where(keep, d * gB + s["D"][:, None] * dy, 0.0).to(dt)
    dd = (A * q).sum(3).view(B, D, T) + x * gB
    draw_ = torch.where(keep, dd / (1 + torch.exp(-raw)), 0.0)
    got["ddelta"] = draw_.to(dt)
    got["ddelta_bias"] = draw_.sum((0, 2))
    got["dA"] = (q * d.view(five)).sum((0, 4)).view(D, N)
    got["dB"] = (g * (d * x).view(five)).sum(2).view(s["B"].shape).to(dt)
    got["dC"] = (h * dy.view(five)).sum(2).view(s["C"].shape).to(dt)
    got["dD"] = (dy * x).sum((0, 2))
    if c["state"]:
        got["dh0"] = (a[..., 0] * g[..., 0]).reshape(B, D, N)
    return got


def _into(pool, slots, new):
    """Writes the rows that are not padding to their places."""
    ok = slots >= 0
    pool[slots[ok]] = new[ok].to(pool.dtype)


def _plain_step(s):
    c = s["case"]
    B, D, N, G = c["B"], c["D"], c["N"], c["G"]
    x, d = s["x"].float(), _softplus(s["delta"].float() + s["delta_bias"])
    Bt, Ct = (s[n].float().view(B, G, 1, N).expand(B, G, D // G, N).reshape(B, D, N) for n in ("B", "C"))
    h = s["state"][s["slots"].clamp(min=0)]
    h = torch.exp(d[..., None] * s["A"]) * h + (d * x)[..., None] * Bt
    y = (Ct * h).sum(-1) + s["D"] * x
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    _into(s["state"], s["slots"], h)
    return dict(y=torch.where(s["slots"][:, None] >= 0, y, 0.0).to(s["x"].dtype), state=s["state"])


def _plain_conv(s):
    c = s["case"]
    B, D, T, K, dt = c["B"], c["D"], c["T"], c["K"], s["x"].dtype
    keep = _inside(s, T)
    w = s["w"]
    x0 = torch.zeros(B, D, K - 1, device="cuda") if s["x0"] is None else s["x0"].float()
    xe = torch.cat([x0, torch.where(keep, s["x"].float(), 0.0)], -1)
    win = xe.unfold(-1, K, 1)                            # (B, D, T, K): the taps of every position
    pre = (win * w[:, None]).sum(-1) + s["b"][:, None]
    got = dict(y=torch.where(keep, _silu(pre) if c["silu"] else pre, 0.0).to(dt))
    n = torch.full((B,), T, device="cuda") if s["lengths"] is None else s["lengths"]
    at = (n[:, None] + torch.arange(K - 1, device="cuda"))[:, None].expand(B, D, K - 1)
    if c["state"]:
        got["last"] = xe.gather(2, at).to(dt)
    if not c["train"]:
        return got
    dpre = torch.where(keep, s["dy"].float(), 0.0)
    if c["silu"]:
        dpre = dpre * _dsilu(pre)
    # position t of the extended input feeds outputs t - K + 1 ... t
    gap = torch.zeros(B, D, K - 1, device="cuda")
    dxe = (torch.cat([gap, dpre, gap], -1).unfold(-1, K, 1) * w.flip(1)[:, None]).sum(-1)
    if c["state"]:
        dxe.scatter_add_(2, at, s["dlast"].float())
        got["dx0"] = dxe[..., :K - 1].to(dt)
    got["dx"] = torch.where(keep, dxe[..., K - 1:], 0.0).to(dt)
    got["dw"] = (win * dpre[..., None]).sum((0, 2))
    got["db"] = dpre.sum((0, 2))
    return got


def _plain_convstep(s):
    c = s["case"]
    x = s["x"]
    win = torch.cat([s["state"][s["slots"].clamp(min=0)], x[..., None]], -1)
    y = (win.float() * s["w"]).sum(-1) + s["b"]
    if c["silu"]:
        y = _silu(y)
    _into(s["state"], s["slots"], win[..., 1:])
    return dict(y=torch.where(s["slots"][:, None] >= 0, y, 0.0).to(x.dtype), state=s["state"])


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return dict(scan=_plain_scan, step=_plain_step, conv=_plain_conv, convstep=_plain_convstep)[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------ work ----


def work(case):
    c = case
    es, BD = (4 if c["dtype"] == "f32" else 2), case["B"] * case["D"]
    if c["op"] == "scan":
        T, N, G = c["T"], c["N"], c["G"]
        row, bc, st = BD * T * es, c["B"] * G * N * T * es, BD * N * 4
        rows = 3 + bool(c["z"])                          # tokens, delta, z in; y out
        small = c["D"] * (N + 2) * 4
        bytes_, flops = rows * row + 2 * bc + small + 2 * st * c["state"], 7 * BD * T * N
        if c["train"]:                                   # dy in; gradients of every input out
            bytes_ += (1 + rows - 1) * row + 2 * bc + small + 2 * st * c["state"]
            flops += 16 * BD * T * N
        return dict(bytes=bytes_, flops=flops)
    if c["op"] == "step":
        return dict(bytes=BD * (c["N"] * 8 + (3 + bool(c["z"])) * es) + 2 * c["B"] * c["G"] * c["N"] * es + c["D"] * (c["N"] + 2) * 4,
                    flops=7 * BD * c["N"])
    K = c["K"]
    small, st = c["D"] * (K + 1) * 4, BD * (K - 1) * es
    if c["op"] == "convstep":
        return dict(bytes=BD * 2 * es + 2 * st + small, flops=2 * BD * K)
    row = BD * c["T"] * es
    bytes_, flops = 2 * row + small + 2 * st * c["state"], 2 * BD * c["T"] * K
    if c["train"]:
        bytes_ += 2 * row + small + 2 * st * c["state"]
        flops += 4 * BD * c["T"] * K
    return dict(bytes=bytes_, flops=flops)


# -------------------------------------------------------------------- from the definition ----


def exact(case, seed):
    """The operators' values in 64 bits, walked one position after the other as they are defined."""
    s = prepare(case, seed)
    c = case
    with torch.no_grad():
        f = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
        return dict(scan=_exact_scan, step=_exact_step, conv=_exact_conv, convstep=_exact_convstep)[c["op"]](c, f)


def _sig(v):
    return torch.sigmoid(v)


def _wide(v, D):
    """(B, [G,] N, ...) as (B, D, N, ...): every channel its group's vector."""
    if v.dim() == 3:
        return v[:, None].expand(-1, D, -1, -1)
    return v.repeat_interleave(D // v.shape[1], dim=1)


def _exact_scan(c, f):
    B, D, T, N = c["B"], c["D"], c["T"], c["N"]
    if T > 20000:
        return None
    n = f["lengths"] if f["lengths"] is not None else torch.full((B,), T, device="cuda")
    live = torch.arange(T, device="cuda")[None, :] < n[:, None]               # (B, T)
    raw = f["delta"] + f["delta_bias"][None, :, None]
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    G = c["G"]
    Bv, Cv = f["B"].reshape(B, G, N, T), f["C"].reshape(B, G, N, T)
    per = D // G
    h = f["h0"].clone() if f["h0"] is not None else torch.zeros(B, D, N, device="cuda", dtype=torch.float64)
    start = h.clone()
    train = c["train"]
    hist = torch.empty(T, B, D, N, device="cuda", dtype=torch.float64) if train else None
    y = torch.zeros(B, D, T, device="cuda", dtype=torch.float64)
    for t in range(T):
        m = live[:, t].view(B, 1, 1)
        d = dt[:, :, t, None]
        b_t = Bv[..., t].repeat_interleave(per, 1)
        c_t = Cv[..., t].repeat_interleave(per, 1)
        h = torch.where(m, torch.exp(d * f["A"]) * h + d * b_t * f["x"][:, :, t, None], h)
        if train:
            hist[t] = h
        y[:, :, t] = torch.where(m[..., 0], (h * c_t).sum(-1) + f["D"] * f["x"][:, :, t], 0.0)
    out = y if f["z"] is None else y * f["z"] * _sig(f["z"])
    got = dict(y=torch.where(live[:, None], out, 0.0))
    if c["state"]:
        got["last"] = h
    if not train:
        return got
    g_out = torch.where(live[:, None], f["dy"], 0.0)
    if f["z"] is None:
        gy = g_out
    else:
        sg = _sig(f["z"])
        gy = g_out * f["z"] * sg
        got["dz"] = g_out * y * (sg + f["z"] * sg * (1 - sg))
    dx, dd = torch.zeros_like(y), torch.zeros_like(y)
    dA = torch.zeros(D, N, device="cuda", dtype=torch.float64)
    dB, dC = torch.zeros_like(Bv), torch.zeros_like(Cv)
    lam = f["dlast"].clone() if c["state"] else torch.zeros_like(h)           # dL/dh_t, flowing back
    for t in range(T - 1, -1, -1):
        m = live[:, t].view(B, 1, 1)
        prev = hist[t - 1] if t else start
        d, xt = dt[:, :, t, None], f["x"][:, :, t, None]
        b_t = Bv[..., t].repeat_interleave(per, 1)
        c_t = Cv[..., t].repeat_interleave(per, 1)
        e = torch.exp(d * f["A"])
        at = lam + c_t * gy[:, :, t, None]
        at = torch.where(m, at, torch.zeros_like(at))
        dC[..., t] = (hist[t] * gy[:, :, t, None] * m).view(B, G, per, N).sum(2)
        dB[..., t] = (at * d * xt).view(B, G, per, N).sum(2)
        dx[:, :, t] = torch.where(m[..., 0], (at * b_t).sum(-1) * dt[:, :, t] + f["D"] * gy[:, :, t], 0.0)
        through = at * e * prev
        dA += (through * d).sum(0)
        dd[:, :, t] = (through * f["A"]).sum(-1) + torch.where(m[..., 0], (at * b_t).sum(-1) * f["x"][:, :, t], 0.0)
        lam = torch.where(m, at * e, lam)
    draw_ = torch.where(live[:, None], dd * _sig(raw), 0.0)
    got.update(dx=dx, ddelta=draw_, ddelta_bias=draw_.sum((0, 2)), dA=dA,
               dB=dB.view(f["B"].shape), dC=dC.view(f["C"].shape),
               dD=torch.where(live[:, None], gy * f["x"], 0.0).sum((0, 2)))
    if c["state"]:
        got["dh0"] = lam
    return got


def _exact_step(c, f):
    state = f["state"].clone()
    y = torch.zeros_like(f["x"])
    bad = f["slots"] < 0
    where = f["slots"].clone()
    where[bad] = 0
    raw = f["delta"] + f["delta_bias"]
    d = torch.logaddexp(raw, torch.zeros_like(raw))
    b, cc = (_wide(v.reshape(c["B"], c["G"], c["N"], 1), c["D"])[..., 0] for v in (f["B"], f["C"]))
    h = state[where] * torch.exp(torch.einsum("bd,dn->bdn", d, f["A"])) + b * (d * f["x"])[..., None]
    y = torch.einsum("bdn,bdn->bd", h, cc) + f["x"] * f["D"]
    if f["z"] is not None:
        y = y * f["z"] * _sig(f["z"])
    y[bad] = 0
    state[where[~bad]] = h[~bad]
    return dict(y=y, state=state)


def _exact_conv(c, f):
    B, D, T, K = c["B"], c["D"], c["T"], c["K"]
    n = f["lengths"] if f["lengths"] is not None else torch.full((B,), T, device="cuda")
    live = (torch.arange(T, device="cuda")[None, :] < n[:, None])[:, None]
    first = f["x0"] if f["x0"] is not None else torch.zeros(B, D, K - 1, device="cuda", dtype=torch.float64)
    ext = torch.cat([first, f["x"] * live], -1)
    pre = f["b"][None, :, None].expand(B, D, T).clone()
    for k in range(K):
        pre += f["w"][None, :, k, None] * ext[..., k:k + T]
    y = pre * _sig(pre) if c["silu"] else pre
    got = dict(y=torch.where(live, y, 0.0))
    ends = n.tolist()
    if c["state"]:
        got["last"] = torch.stack([ext[i, :, e:e + K - 1] for i, e in enumerate(ends)])
    if not c["train"]:
        return got
    sg = _sig(pre)
    dp = f["dy"] * live * ((sg + pre * sg * (1 - sg)) if c["silu"] else 1.0)
    dext = torch.zeros_like(ext)
    dw = torch.empty(D, K, device="cuda", dtype=torch.float64)
    for k in range(K):
        dext[..., k:k + T] += f["w"][None, :, k, None] * dp
        dw[:, k] = (dp * ext[..., k:k + T]).sum((0, 2))
    if c["state"]:
        for i, e in enumerate(ends):
            dext[i, :, e:e + K - 1] += f["dlast"][i]
        got["dx0"] = dext[..., :K - 1]
    got.update(dx=torch.where(live, dext[..., K - 1:], 0.0), dw=dw, db=dp.sum((0, 2)))
    return got


def _exact_convstep(c, f):
    K = c["K"]
    state, bad = f["state"].clone(), f["slots"] < 0
    where = f["slots"].clone()
    where[bad] = 0
    old = state[where]
    y = f["b"] + f["x"] * f["w"][:, K - 1]
    for k in range(K - 1):
        y = y + old[..., k] * f["w"][:, k]
    if c["silu"]:
        y = y * _sig(y)
    y[bad] = 0
    state[where[~bad]] = torch.cat([old[~bad][..., 1:], f["x"][~bad][..., None]], -1)
    return dict(y=y, state=state)
