"""The contrastive loss over the feature bank (linear, log_probs, bank_log_probs) against plain formulas in 64 bits.

Tolerances are bounds, element by element, from the arithmetic that the kernels are allowed: u = 2^-24 is half a step of f32, u_T = eps / 2 half a
step of the tensor's type.  A sum of n products in f32 is off by at most (n + 2) u times the sum of their magnitudes, whatever its order."""
import ctypes as C
import math

import pytest
import torch

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = float("inf")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step among the subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def within(got, want, bound, what):
    """Same infinities, NaN in the same places, everything else within the bound."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, what
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), f"{what}: other infinities"
    err = (got - want).abs()[fin]
    lim = (bound if torch.is_tensor(bound) else torch.full_like(want, bound)).double().expand_as(want)[fin]
    bad = ~(err <= lim)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst {float((err / lim.clamp(min=1e-300)).max()):.3g} times"


# ---- linear ---------------------------------------------------------------------------------------------------------
ACT = {"none": lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}
# largest slope, largest second derivative (gelu: 2 / sqrt(2 pi) at 0; silu: 1/2 at 0)
SLOPE = {"none": 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1}
CURVE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5}


def linear_bounds(x, w, b, r, g, act, alpha, beta, dtype):
    """-> (values, bounds): y and the gradients in 64 bits with what the kernels may be off."""
    X, W = x.double(), w.double()
    Bv = b.double() if b is not None else torch.zeros(w.shape[0], dtype=torch.float64, device=x.device)
    R = r.double() if r is not None else torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    G, uT, t = g.double(), half_step(dtype), tiny(dtype)
    K, N, M = x.shape[1], w.shape[0], x.shape[0]
    z = (alpha * (X @ W.T) + Bv).requires_grad_()
    a = ACT[act](z)
    (slope,) = torch.autograd.grad(a.sum(), z)
    z, a = z.detach(), a.detach()
    y = a + beta * R
    mag = abs(alpha) * (X.abs() @ W.abs().T) + Bv.abs()
    z_err = (K + 4) * U * mag
    # the activation itself: a few steps of its argument's and value's size
    y_err = SLOPE[act] * z_err + 8 * U * (z.abs() + a.abs() + abs(beta) * R.abs())
    dz = G * slope
    pre_err = z_err + (0.0 if act == "none" else uT) * z.abs() + t
    s_err = CURVE[act] * pre_err + (0.0 if act in ("none", "relu") else 16 * U * (1 + z.abs()))
    if act == "relu":
        s_err = s_err + (z.abs() <= z_err).double()                    # the sign of a value within its error is open
    dz_exact_err = G.abs() * s_err                                     # before dz is rounded to its type
    dz_err = dz_exact_err + (0.0 if act == "none" else uT) * (dz.abs() + dz_exact_err) + t
    dx, dw, db = alpha * dz @ W, alpha * dz.T @ X, dz.sum(0)
    dx_err = abs(alpha) * (dz_err @ W.abs() + (N + 4) * U * (dz.abs() + dz_err) @ W.abs())
    dw_err = abs(alpha) * (dz_err.T @ X.abs() + (M + 4) * U * (dz.abs() + dz_err).T @ X.abs())
    db_err = dz_exact_err.sum(0) + (M + 4) * U * (dz.abs() + dz_exact_err).sum(0)
    vals = {"y": y, "x": dx, "weight": dw, "bias": db, "residual": beta * G}
    errs = {"y": y_err, "x": dx_err, "weight": dw_err, "bias": db_err, "residual": 2 * U * (beta * G).abs()}
    return vals, {k: e + uT * (vals[k].abs() + e) + t for k, e in errs.items()}


def linear_case(dev, M, N, K, dtype, act, bias=True, residual=True, alpha=0.5, beta=-1.5, seed=0):
    import nemo_amd
    gen = torch.Generator(device=dev).manual_seed(seed)
    def rnd(*s, std=1.0):
        return (torch.randn(*s, generator=gen, device=dev) * std).to(dtype)
    x, w = rnd(M, K), rnd(N, K, std=max(K, 1) ** -0.5)
    b, r, g = rnd(N) if bias else None, rnd(M, N) if residual else None, rnd(M, N)
    leaves = {k: v.requires_grad_() for k, v in (("x", x), ("weight", w), ("bias", b), ("residual", r)) if v is not None}
    y = nemo_amd.linear(x, w, b, r, act, alpha, beta)
    assert y.dtype == dtype and y.shape == (M, N)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), g)))
    d = {k: v.detach() for k, v in leaves.items()}
    vals, bounds = linear_bounds(d["x"], d["weight"], d.get("bias"), d.get("residual"), g, act, alpha, beta, dtype)
    within(y, vals["y"], bounds["y"], "y")
    for k, v in grads.items():
        assert v.dtype == dtype
        within(v, vals[k], bounds[k], f"gradient of {k}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 129, 64), (2, 1000, 4096), (3, 5, 7), (16, 48, 33), (17, 64, 640), (64, 512, 256), (65, 130, 200),
                                   (128, 128, 128), (129, 257, 100), (1000, 72, 515), (4097, 40, 24), (300, 700, 1024)])
def test_linear_sizes(gpu, M, N, K, dtype):
    linear_case(gpu, M, N, K, TYPES[dtype], "none" if (M + N) % 2 else "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,N,K", [(32, 300, 512), (33, 1000, 2100), (900, 50, 300), (5000, 700, 1030), (6000, 2000, 100), (7900, 2049, 70)])
def test_linear_every_tile(gpu, M, N, K, dtype):
    """Sizes for which the products of the three directions take tiles of 32, 64, 128 and 256 rows, with and without splits."""
    linear_case(gpu, M, N, K, TYPES[dtype], "silu", residual=(M % 2 == 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
def test_linear_epilogues(gpu, act, bias, residual, dtype):
    linear_case(gpu, 130, 68, 96, TYPES[dtype], act, bias, residual)
    linear_case(gpu, 9, 33, 65, TYPES[dtype], act, bias, residual, alpha=1.0, beta=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_nothing_to_sum_or_to_write(gpu, dtype):
    import nemo_amd
    dt = TYPES[dtype]
    for M, N, K in ((0, 5, 4), (5, 0, 4), (5, 3, 0), (0, 0, 0)):
        x, w = torch.ones(M, K, device=gpu, dtype=dt, requires_grad=True), torch.ones(N, K, device=gpu, dtype=dt, requires_grad=True)
        b = torch.full((N,), -2.0, device=gpu, dtype=dt, requires_grad=True)
        r = torch.full((M, N), 3.0, device=gpu, dtype=dt, requires_grad=True)
        for act, want in (("none", 1.0), ("relu", 3.0)):
            y = nemo_amd.linear(x, w, b, r, act)
            assert y.shape == (M, N) and torch.equal(y, torch.full_like(y, want))
            gx, gw, gb, gr = torch.autograd.grad(y, (x, w, b, r), torch.ones_like(y))
            assert not gx.any() and not gw.any() and torch.equal(gr, torch.ones_like(gr))
            assert torch.equal(gb, torch.full_like(gb, float(M) if act == "none" else 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_strides_and_starts(gpu, dtype):
    """Slices of wider rows, rows that start at any element, transposed and expanded views, more leading dimensions."""
    import nemo_amd
    dt = TYPES[dtype]
    gen = torch.Generator(device=gpu).manual_seed(5)
    big = torch.randn(3, 50, 401, generator=gen, device=gpu).to(dt)
    wide = torch.randn(70, 409, generator=gen, device=gpu).to(dt)
    g = torch.randn(3, 50, 70, generator=gen, device=gpu).to(dt)
    for x, w, r in ((big[:, :, 1:97], wide[:, 3:99], None),
                    (big[..., :96], wide[:, 8:104], wide[:50, :70].expand(3, 50, 70)),
                    (big.permute(1, 0, 2)[..., :64].transpose(0, 1), wide.T[:64].T, big[:, :, 2:72]),
                    (big[:, :, ::2][..., :128], wide[:, ::3][:, :128], big[..., 100:170])):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = nemo_amd.linear(x, w, None, r, "silu", 0.25, 2.0)
        assert y.shape == (3, 50, 70)
        gx, gw = torch.autograd.grad(y, (x, w), g)
        K = x.shape[-1]
        vals, bounds = linear_bounds(x.detach().reshape(150, K), w.detach(), None, None if r is None else r.reshape(150, 70), g.reshape(150, 70), "silu",
                                     0.25, 2.0, dt)
        within(y.reshape(150, 70), vals["y"], bounds["y"], "y")
        within(gx.reshape(150, K), vals["x"], bounds["x"], "gradient of x")
        within(gw, vals["weight"], bounds["weight"], "gradient of weight")
    # a gradient that arrives expanded
    x, w = big[0, :, :96].detach().requires_grad_(), wide[:, :96].detach().requires_grad_()
    (gx,) = torch.autograd.grad(nemo_amd.linear(x, w).sum(), x)
    vals, bounds = linear_bounds(x.detach(), w.detach(), None, None, torch.ones(50, 70, device=gpu, dtype=dt), "none", 1.0, 1.0, dt)
    within(gx, vals["x"], bounds["x"], "gradient of x from a sum")


@pytest.mark.gpu
def test_linear_infinities_and_nan(gpu):
    """Non-finite inputs reach the outputs they are a term of, and no others."""
    import nemo_amd
    for dt in TYPES.values():
        x = torch.ones(70, 40, device=gpu, dtype=dt)
        w = torch.ones(90, 40, device=gpu, dtype=dt)
        x[3, 39], x[69, 0], w[89, 5] = INF, float("nan"), -INF
        y = nemo_amd.linear(x, w)
        want = x.double() @ w.double().T
        within(y, want, half_step(dt) * want.abs(), "y")
        assert torch.isinf(y[3, 0]) and torch.isnan(y[3, 89]) and torch.isnan(y[69]).all() and bool(torch.isfinite(y[:3, :89]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_linear_gradient_against_differences(gpu, act):
    """Along random directions in f32: (L(+h) - L(-h)) / 2h of the kernel's own values, L = sum g y summed in 64 bits.  The values are off by y_err each
    (linear_bounds), so the quotient by sum |g| y_err / h; the third derivative adds h^2 / 6 times at most 1.7 |g| |dz|^3 (gelu and silu)."""
    import nemo_amd
    M, N, K, h = 33, 20, 48, 0.02
    gen = torch.Generator(device=gpu).manual_seed(3)
    x, w, b = (torch.randn(*s, generator=gen, device=gpu) * f for s, f in (((M, K), 1.0), ((N, K), 0.15), ((N,), 1.0)))
    vx, vw, vb = (torch.randn(t.shape, generator=gen, device=gpu) * f for t, f in ((x, 0.2), (w, 0.03), (b, 0.2)))
    g = torch.randn(M, N, generator=gen, device=gpu)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(nemo_amd.linear(*leaves, activation=act), leaves, g)
    slope = sum(float((gr.double() * v.double()).sum()) for gr, v in zip(grads, (vx, vw, vb)))
    L = [float((nemo_amd.linear(x + s * h * vx, w + s * h * vw, b + s * h * vb, activation=act).double() * g.double()).sum()) for s in (1, -1)]
    _, bounds = linear_bounds(x, w, b, None, g, act, 1.0, 1.0, torch.float32)
    dz = (vx.double().abs() @ w.double().abs().T + x.double().abs() @ vw.double().abs().T + vb.double().abs() + h * vx.double().abs() @ vw.double().abs().T)
    # second-order terms of z itself (x and w move together): z'' = 2 vx vw^T enters with the slope's curvature
    zz = 2 * vx.double().abs() @ vw.double().abs().T
    third = (g.double().abs() * (1.7 * dz ** 3 + 3 * CURVE[act] * dz * zz)).sum()
    # the inputs x +- h v are rounded to f32 too: half a step of theirs moves L by at most u (|grad| |x|)
    moved = sum(float((gr.double().abs() * t.double().abs()).sum()) for gr, t in zip(grads, (x, w, b))) * 2 * U / h
    lim = float((g.double().abs() * bounds["y"]).sum()) / h + h * h / 6 * float(third) + moved
    assert abs((L[0] - L[1]) / (2 * h) - slope) <= lim
    assert lim < 0.2 * abs(slope) or abs(slope) < 1.0          # the bound says something


@pytest.mark.gpu
def test_linear_refusals(gpu):
    import nemo_amd
    x, w = torch.zeros(4, 8, device=gpu), torch.zeros(5, 8, device=gpu)
    for bad in (lambda: nemo_amd.linear(x, torch.zeros(5, 7, device=gpu)), lambda: nemo_amd.linear(x, w[0]),
                lambda: nemo_amd.linear(x, w, bias=torch.zeros(4, device=gpu)), lambda: nemo_amd.linear(x, w, residual=torch.zeros(5, device=gpu)),
                lambda: nemo_amd.linear(x, w, activation="tanh"), lambda: nemo_amd.linear(x, w, alpha=float("nan"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: nemo_amd.linear(x, w.half()), lambda: nemo_amd.linear(x.double(), w.double()), lambda: nemo_amd.linear(x, w, bias=3.0)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="CPU"):
        nemo_amd.linear(x, w.cpu())
    y = nemo_amd.linear(x.requires_grad_(), w.requires_grad_(), activation="silu")
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()                                            # differentiable once


# ---- log probabilities -----------------------------------------------------------------------------------------------
def probs_reference(z, targets, top, g=None):
    """In 64 bits from scores z (-inf: left out) -> dict of values; with g = (g_logp, g_entropy, g_lse) also dz."""
    S, V = z.shape
    if V == 0:
        z, V = torch.full((S, 1), -INF, dtype=torch.float64, device=z.device), 0
    nothing = (z == -INF).all(1)
    lse = torch.logsumexp(z, 1)
    broken = torch.isnan(lse) | (lse == INF)
    lse = torch.where(broken, torch.full_like(lse, float("nan")), lse)
    peak = z.amax(1, keepdim=True).clamp(min=-torch.finfo(torch.float64).max)
    log_s = torch.logsumexp(z - peak, 1, keepdim=True)                 # z - lse would lose log s next to scores of 1e38
    lp = torch.where(z == -INF, z, (z - peak) - log_s)
    p = torch.where(z == -INF, torch.zeros_like(z), lp.exp())
    ent = torch.where(nothing, torch.zeros_like(lse), -torch.where(p > 0, p * lp, p * 0).sum(1) + torch.where(broken, lse, torch.zeros_like(lse)))
    inside = (targets >= 0) & (targets < V)
    at = targets.clamp(0, max(V - 1, 0))
    logp = torch.where(targets == -1, torch.zeros_like(lse), torch.full_like(lse, float("nan")))
    picked = lp.gather(1, at[:, None])[:, 0]
    logp = torch.where(inside, torch.where(broken, lse, picked), logp)
    out = {"logp": logp, "entropy": ent, "lse": lse}
    if top:
        zs = torch.where(torch.isnan(z), torch.full_like(z, -INF), z)
        val, idx = torch.sort(zs, dim=1, descending=True, stable=True)
        val, idx = val[:, :top], idx[:, :top]
        if val.shape[1] < top:
            pad = top - val.shape[1]
            val, idx = torch.nn.functional.pad(val, (0, pad), value=-INF), torch.nn.functional.pad(idx, (0, pad), value=-1)
        gone = (val == -INF) | broken[:, None]
        out["top_index"] = torch.where(gone, torch.full_like(idx, -1), idx)
        out["top_logp"] = torch.where(broken[:, None], lse[:, None].expand_as(val), torch.where(val == -INF, val, (val - peak) - log_s))
    if g is not None:
        gl, gh, gs = (torch.zeros_like(lse) if t is None else t.double() for t in g)
        gl = torch.where(inside, gl, torch.zeros_like(gl))
        dz = p * (gs - gl)[:, None] - torch.where(p > 0, p * gh[:, None] * (lp + ent[:, None]), p * 0)
        dz = dz.scatter_add(1, at[:, None], torch.where(inside, gl, torch.zeros_like(gl))[:, None])
        dz = torch.where((targets < -1) | (targets >= V), torch.full_like(gl, float("nan")), torch.zeros_like(gl))[:, None] + dz
        dz = torch.where(z == -INF, torch.zeros_like(dz), dz)
        out["dz"] = dz
        out["p"] = p
    return out


def probs_bounds(ref, z, z_err, V, g=None):
    """What the statistics may be off where scores are off by z_err [S] (absolute).  With D = the largest |z| of a row whose probability counts:
    exp(z - m) is off relatively by 2 z_err (z and m) + (1.45 |z - m| + 4) u (the product with log2 e, the hardware's exponential), and
    |z - m| <= 2 D; rescalings when the maximum moves add as much again; a sum of V terms, at most V / 64 + 40 additions in a row (a lane's
    own, lanes, parts), (V / 64 + 40) u.  logp = (z_t - m) - log s: besides lse's error that of z_t itself, which may be far from the others (a
    weight of 1e5): a product, a difference and two more differences of magnitudes up to |z_t| <= |logp| + |lse|, 4 u of them."""
    D = torch.where(torch.isfinite(z) & (ref["p"] > 1e-40) if "p" in ref else torch.isfinite(z), z.abs(), torch.zeros_like(z))
    D = D.amax(1) if z.shape[1] else torch.zeros(z.shape[0], dtype=torch.float64, device=z.device)
    rel = 2 * z_err + (8 * D + V / 64 + 60) * U
    D1 = D + 1
    out = {"lse": rel + 4 * U * D1, "logp": 2 * rel + 8 * U * D1, "entropy": (2 * D1 + 2) * rel + 8 * U * D1}
    far = lambda t: 4 * U * torch.where(torch.isfinite(t), t.abs(), torch.zeros_like(t))
    out["top_logp"] = out["logp"][:, None] + (far(ref["top_logp"]) if "top_logp" in ref else 0)
    out["logp"] = out["logp"] + far(ref["logp"])
    if g is not None:
        gl, gh, gs = (torch.zeros_like(rel) if t is None else t.double().abs() for t in g)
        lp = torch.where(ref["p"] > 0, ref["p"].clamp(min=1e-300).log().abs(), torch.zeros_like(z))
        size = (gl + gs)[:, None] + gh[:, None] * (lp + ref["entropy"].abs()[:, None] + 1)
        out["dz"] = torch.where(z == -INF, torch.zeros_like(z), 4 * (rel + 4 * U)[:, None] * ref["p"] * size + 4 * U * gl[:, None] + 1e-37)
    return out


def check_probs(got, ref, bounds, top):
    for k in ("logp", "entropy", "lse"):
        assert getattr(got, k).dtype == torch.float32
        within(getattr(got, k), ref[k], bounds[k], k)
    if top:
        assert torch.equal(got.top_index, ref["top_index"]), "best entries"
        within(got.top_logp, ref["top_logp"], bounds["top_logp"], "top_logp")
    else:
        assert got.top_logp is None and got.top_index is None


def scores64(raw, scale, weights):
    z = raw.double() * scale
    if weights is None:
        return z
    w = weights.double().expand_as(z)
    gone = w == INF
    return torch.where(gone, torch.full_like(z, -INF), z - torch.where(gone, torch.zeros_like(w), w))


def make_weights(kind, S, V, gen, dev):
    if kind == "none":
        return None
    w = torch.rand(*((V,) if kind == "bank" else (S, V)), generator=gen, device=dev).mul_(4).floor_()
    w[torch.rand(w.shape, generator=gen, device=dev) < 0.2] = INF
    w[torch.rand(w.shape, generator=gen, device=dev) < 0.1] = 1.0e5
    return w


def upstream(S, gen, dev, which="logp entropy lse"):
    return tuple(torch.randn(S, generator=gen, device=dev) if k in which.split() else None for k in ("logp", "entropy", "lse"))


def run_grads(r, g, leaves):
    outs = [(o, t) for o, t in zip((r.logp, r.entropy, r.lse), g) if t is not None]
    return torch.autograd.grad([o for o, _ in outs], leaves, [t for _, t in outs])


def log_probs_case(dev, S, V, dtype, kind, top, scale=0.5, which="logp entropy lse", seed=0):
    import nemo_amd
    gen = torch.Generator(device=dev).manual_seed(seed)
    logits = (torch.randint(-3000, 3000, (S, V), generator=gen, device=dev) / 512).to(dtype).requires_grad_()     # many ties in 16 bits
    weights = make_weights(kind, S, V, gen, dev)
    targets = torch.randint(-1, max(V, 1), (S,), generator=gen, device=dev) if V else torch.full((S,), -1, device=dev)
    g = upstream(S, gen, dev, which)
    r = nemo_amd.log_probs(logits, targets, weights, scale, top)
    z = scores64(logits.detach(), scale, weights)
    # best entries and ties go by the scores in 32 bits
    z32 = logits.detach().float() * scale
    if weights is not None:
        z32 = torch.where(weights == INF, torch.full_like(z32, -INF), z32 - weights)
    ref = probs_reference(z, targets, top, g)
    if top:
        ref["top_index"] = probs_reference(z32.double(), targets, top)["top_index"]
        ref["top_logp"] = torch.where(ref["top_index"] < 0, torch.full_like(ref["top_logp"], -INF),
                                      (z - ref["lse"][:, None]).gather(1, ref["top_index"].clamp(min=0)) if V else ref["top_logp"])
    z_err = 2 * U * torch.where(torch.isfinite(z) & (ref["p"] > 1e-40), z.abs() + (0 if weights is None else 8.0), torch.zeros_like(z)).amax(1) if V \
        else torch.zeros(S, dtype=torch.float64, device=dev)
    if weights is not None and V:
        # a finite weight of 1e5 rounds the score to its own steps; such places count only where a row has nothing else
        z_err = z_err + 2 * U * torch.where(ref["p"] > 1e-40, torch.where(torch.isfinite(weights), weights, torch.zeros_like(weights)).double().expand_as(z),
                                            torch.zeros_like(z)).amax(1)
    bounds = probs_bounds(ref, z, z_err, V, g)
    check_probs(r, ref, bounds, top)
    (gx,) = run_grads(r, g, [logits])
    assert gx.dtype == dtype and gx.shape == (S, V)
    want = scale * ref["dz"][:, :V]
    b = abs(scale) * bounds["dz"][:, :V]
    within(gx, want, b + half_step(dtype) * (want.abs() + b) + tiny(dtype) * 2 * (want != 0), "gradient of logits")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["none", "bank", "rows"])
@pytest.mark.parametrize("S,V", [(1, 1), (1, 7), (2, 64), (5, 1118), (3, 1031), (70, 2049), (1, 40003), (3, 70001), (2500, 33), (1100, 1500)])
def test_log_probs_sizes(gpu, S, V, kind, dtype):
    log_probs_case(gpu, S, V, TYPES[dtype], kind, 0 if V % 2 else 5)
    log_probs_case(gpu, S, V, TYPES[dtype], kind, 16 if V % 2 else 1, seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["logp", "entropy", "lse", "logp lse"])
def test_log_probs_single_gradients(gpu, which):
    log_probs_case(gpu, 40, 301, torch.float32, "rows", 0, which=which)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-2.0, 0.0, 1e-35, 50.0])
@pytest.mark.parametrize("kind", ["none", "rows"])
def test_log_probs_scales(gpu, kind, scale):
    log_probs_case(gpu, 30, 1500, torch.float32, kind, 0 if scale == 1e-35 else 5, scale=scale)
    log_probs_case(gpu, 1100, 700, torch.bfloat16, kind, 0, scale=scale)


@pytest.mark.gpu
def test_gradients_of_some_inputs_only(gpu):
    """One input at a time needs a gradient; gradients come from sums (expanded, stride 0); weights are one row expanded."""
    import nemo_amd
    gen = torch.Generator(device=gpu).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=gpu)
    args = {"x": rnd(60, 70), "weight": rnd(90, 70), "bias": rnd(90), "residual": rnd(60, 90)}
    full = {k: v.clone().requires_grad_() for k, v in args.items()}
    want = dict(zip(full, torch.autograd.grad(nemo_amd.linear(**full, activation="silu", beta=0.5).sum(), list(full.values()))))
    for k in args:
        leaf = args[k].clone().requires_grad_()
        (got,) = torch.autograd.grad(nemo_amd.linear(**{**args, k: leaf}, activation="silu", beta=0.5).sum(), leaf)
        assert torch.equal(got, want[k]), k
    f, b, t, w = rnd(60, 32), rnd(90, 32), torch.randint(0, 90, (60,), generator=gen, device=gpu), torch.rand(1, 90, generator=gen, device=gpu)
    F, B = f.clone().requires_grad_(), b.clone().requires_grad_()
    r = nemo_amd.bank_log_probs(F, B, t, w.expand(60, 90), scale=0.3)
    wf, wb = torch.autograd.grad(r.logp.sum(), (F, B), retain_graph=True)
    assert torch.equal(torch.autograd.grad(nemo_amd.bank_log_probs(F, b, t, w[0], scale=0.3).logp.sum(), F)[0], wf)
    assert torch.equal(torch.autograd.grad(nemo_amd.bank_log_probs(f, B, t, w.expand(60, 90).contiguous(), scale=0.3).logp.sum(), B)[0], wb)
    assert torch.equal(torch.autograd.grad(r.logp.sum(), B)[0], wb)


def special_rows(dev):
    """Rows of 300 scores (f32) and targets: what a mask, an infinity or a NaN may leave."""
    V, nan = 300, float("nan")
    gen = torch.Generator(device=dev).manual_seed(9)
    base = torch.randn(V, generator=gen, device=dev)
    rows, weights, targets = [], [], []

    def add(logit, weight, target):
        rows.append(logit)
        weights.append(weight)
        targets.append(target)
    zero, allgone = torch.zeros(V, device=dev), torch.full((V,), INF, device=dev)
    add(base, zero, 5)                                               # ordinary
    add(base, allgone, 5)                                            # nothing left
    add(base, allgone, -1)
    add(torch.full((V,), nan, device=dev), allgone, 7)               # NaN only where nothing counts
    one = allgone.clone()
    one[123] = 0
    add(base, one, 123)                                              # one place left
    add(base, one, 5)                                                # the target itself left out
    hidden = base.clone()
    hidden[:120], hidden[124:200], hidden[200:] = nan, INF, -INF
    hidden[120:124] = torch.tensor([1.0, 2.0, 2.0, 3.0], device=dev)
    few = allgone.clone()
    few[120:124] = 0
    add(hidden, few, 121)                                            # infinities and NaN in places left out
    add(torch.where(torch.arange(V, device=dev) == 17, nan, base), zero, 5)      # NaN that counts
    add(torch.where(torch.arange(V, device=dev) == 17, INF, base), zero, 5)      # infinity that counts
    add(torch.where(torch.arange(V, device=dev) < 290, -INF, base), zero, 295)   # most logits -inf
    add(torch.full((V,), -INF, device=dev), zero, 3)
    add(base, torch.full((V,), 3.0e38, device=dev), 4)               # the type's lowest values everywhere
    add(torch.where(torch.arange(V, device=dev) < 150, -3.4028234663852886e38, base), zero, 200)
    add(torch.where(torch.arange(V, device=dev) == 9, 3.0e38, base), zero, 9)
    add(torch.full((V,), 2.5, device=dev), zero, 299)                # all equal
    add(base, zero, -1)
    add(base, zero, 300)                                             # targets outside
    add(base, zero, -2)
    return torch.stack(rows), torch.stack(weights), torch.tensor(targets, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 5])
def test_log_probs_rows_that_masks_leave(gpu, top):
    import nemo_amd
    logits, weights, targets = special_rows(gpu)
    g = upstream(len(targets), torch.Generator(device=gpu).manual_seed(2), gpu)
    leaf = logits.clone().requires_grad_()
    r = nemo_amd.log_probs(leaf, targets, weights, 1.0, top)
    # the scores as 32-bit operations give them: a lowest value less a weight stays what it rounds to
    z = torch.where(weights == INF, torch.full_like(logits, -INF), logits - weights).double()
    ref = probs_reference(z, targets, top, g)
    bounds = probs_bounds(ref, torch.where(z.abs() < 1e30, z, torch.zeros_like(z)), torch.zeros(len(targets), device=gpu, dtype=torch.float64), 300, g)
    bounds["lse"] = bounds["lse"] + 4 * U * torch.where(torch.isfinite(ref["lse"]), ref["lse"].abs(), torch.zeros_like(ref["lse"]))
    check_probs(r, ref, bounds, top)
    (gx,) = run_grads(r, g, [leaf])
    b = bounds["dz"]
    within(gx, ref["dz"], torch.nan_to_num(b + U * (ref["dz"].abs() + b)), "gradient")
    assert not gx[1:4].any() and bool(torch.isfinite(gx[6]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("V", [300, 5000, 20001])
def test_log_probs_extreme_scores(gpu, V, top):
    """Without weights: masks of -inf and of the lowest value, scores up to the type's largest, infinities and NaN that count."""
    import nemo_amd
    gen = torch.Generator(device=gpu).manual_seed(V)
    base, at = torch.randn(V, generator=gen, device=gpu), torch.arange(V, device=gpu)
    full = lambda v: torch.full((V,), v, device=gpu)
    low = -3.4028234663852886e38
    rows = [base, full(-INF), torch.where(at < V - 7, -INF, base), torch.where(at % 2 == 0, -INF, base), full(low), torch.where(at < V - 7, low, base),
            full(-2.0e38), torch.where(at == 9, 3.0e38, base), full(2.5e38), torch.where(at == 17, float("nan"), base), torch.where(at == V - 1, INF, base),
            full(1.0e5), full(-1.0e5), 1.0e4 + 8 * torch.round(base), torch.where(at == 3, -1.0e38, full(-3.0e38))]
    logits = torch.stack(rows)
    S = len(rows)
    targets = torch.full((S,), V - 3, device=gpu)
    targets[1], targets[7], targets[14] = 5, 9, 3
    g = upstream(S, gen, gpu)
    leaf = logits.clone().requires_grad_()
    r = nemo_amd.log_probs(leaf, targets, top=top)
    z = logits.double()
    ref = probs_reference(z, targets, top, g)
    bounds = probs_bounds(ref, torch.where(z.abs() < 1e30, z, torch.zeros_like(z)), torch.zeros(S, device=gpu, dtype=torch.float64), V, g)
    bounds["lse"] = bounds["lse"] + 4 * U * torch.where(torch.isfinite(ref["lse"]), ref["lse"].abs(), torch.zeros_like(ref["lse"]))
    check_probs(r, ref, bounds, top)
    (gx,) = run_grads(r, g, [leaf])
    within(gx, ref["dz"], torch.nan_to_num(bounds["dz"] + U * (ref["dz"].abs() + bounds["dz"])), "gradient")
    assert not gx[1].any()


@pytest.mark.gpu
def test_log_probs_empty_shapes(gpu):
    import nemo_amd
    for fn in (lambda S, V, top: nemo_amd.log_probs(torch.zeros(S, V, device=gpu), torch.full((S,), -1, device=gpu), top=top),
               lambda S, V, top: nemo_amd.bank_log_probs(torch.zeros(S, 16, device=gpu), torch.zeros(V, 16, device=gpu),
                                                         torch.full((S,), -1, device=gpu), top=top)):
        for S, V in ((0, 5), (0, 0), (3, 0)):
            r = fn(S, V, 2)
            assert r.logp.shape == (S,) and r.top_index.shape == (S, 2)
            assert torch.equal(r.lse, torch.full((S,), -INF, device=gpu)) and not r.logp.any() and not r.entropy.any()
            assert torch.equal(r.top_index, torch.full((S, 2), -1, device=gpu)) and torch.equal(r.top_logp, torch.full((S, 2), -INF, device=gpu))


@pytest.mark.gpu
def test_log_probs_strides_starts_and_index_types(gpu):
    import nemo_amd
    gen = torch.Generator(device=gpu).manual_seed(4)
    wide = torch.randn(40, 700, generator=gen, device=gpu)
    ww = torch.rand(40, 900, generator=gen, device=gpu)
    t = torch.randint(0, 333, (80,), generator=gen, device=gpu)[::2]
    for dt in TYPES.values():
        for off in (0, 1, 3, 8):
            src = wide.to(dt)
            a = nemo_amd.log_probs(src[:, off:off + 333], t, ww[:, off + 1:off + 334], top=3)
            b = nemo_amd.log_probs(src[:, off:off + 333].contiguous(), t.contiguous().int(), ww[:, off + 1:off + 334].contiguous(), top=3)
            for p, q in zip(a, b):
                assert torch.equal(p, q)
    c = nemo_amd.log_probs(wide.T[:333].T, t.cpu(), ww[0, ::2][:333], top=3)
    d = nemo_amd.log_probs(wide[:, :333].contiguous(), t, ww[0, ::2][:333].contiguous(), top=3)
    assert all(torch.equal(p, q) for p, q in zip(c, d))


@pytest.mark.gpu
def test_log_probs_refusals(gpu):
    import nemo_amd
    x, t = torch.zeros(4, 9, device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu)
    f, b = torch.zeros(4, 16, device=gpu), torch.zeros(9, 16, device=gpu)
    for call in (lambda **k: nemo_amd.log_probs(k.pop("x", x), k.pop("t", t), **k),
                 lambda **k: nemo_amd.bank_log_probs(f, b, k.pop("t", t), **k)):
        for bad in (dict(t=t[:3]), dict(t=t.cpu() + 9), dict(t=t.cpu() - 2), dict(weights=torch.zeros(4, 8, device=gpu)), dict(top=17), dict(top=-1),
                    dict(top=1.5), dict(scale=INF), dict(weights=torch.zeros(9, device=gpu, requires_grad=True))):
            with pytest.raises(ValueError):
                call(**bad)
        for bad in (dict(t=t.float()), dict(weights=torch.zeros(9, device=gpu).half()), dict(scale=torch.ones((), device=gpu))):
            with pytest.raises(TypeError):
                call(**bad)
        with pytest.raises(RuntimeError):
            call(weights=torch.zeros(9))
    with pytest.raises(ValueError):
        nemo_amd.log_probs(x[0], t)
    with pytest.raises(ValueError, match="256"):
        nemo_amd.bank_log_probs(torch.zeros(4, 300, device=gpu), torch.zeros(9, 300, device=gpu), t)
    with pytest.raises(TypeError):
        nemo_amd.bank_log_probs(f.half(), b.half(), t)
    with pytest.raises(TypeError):
        nemo_amd.bank_log_probs(f, b.bfloat16(), t)


# ---- straight from features and bank -----------------------------------------------------------------------------------
def bank_case(dev, S, V, ch, dtype, kind, top, scale=4.0, which="logp entropy lse", seed=0, features=None, bank=None, weights="make", targets=None):
    import nemo_amd
    gen = torch.Generator(device=dev).manual_seed(seed)
    if features is None:
        # with `top`: on a grid, so that dot products are exact in 32 bits and the order of the best entries is that of 64 bits
        grid = (lambda t: torch.round(t * 128) / 128) if top else (lambda t: t)
        unit = lambda *s: grid(torch.nn.functional.normalize(torch.randn(*s, generator=gen, device=dev), dim=1))
        features, bank = unit(S, ch).to(dtype), unit(V, ch).to(dtype)
    if isinstance(weights, str):
        weights = make_weights(kind, S, V, gen, dev)
    if targets is None:
        targets = torch.randint(-1, V, (S,), generator=gen, device=dev)
    f, b = features.detach().requires_grad_(), bank.detach().requires_grad_()
    g = upstream(S, gen, dev, which)
    r = nemo_amd.bank_log_probs(f, b, targets, weights, scale, top)
    F, Bk = f.detach().double(), b.detach().double()
    raw = F @ Bk.T
    z = scores64(raw, scale, weights)
    ref = probs_reference(z, targets, top, g)
    size = abs(scale)
    mag = size * (torch.nan_to_num(F, 0, 0, 0).abs() @ torch.nan_to_num(Bk, 0, 0, 0).abs().T)
    live = ref["p"] > 1e-40
    fw = 0.0 if weights is None else torch.where(torch.isfinite(weights), weights, torch.zeros_like(weights)).double()
    z_err = torch.where(live, (ch + 4) * U * mag + 2 * U * (mag + fw), torch.zeros_like(z)).amax(1)
    bounds = probs_bounds(ref, z, z_err, V, g)
    check_probs(r, ref, bounds, top)
    gf, gb = run_grads(r, g, [f, b])
    assert gf.dtype == gb.dtype == dtype
    Fc, Bc = torch.nan_to_num(F, 0, 0, 0), torch.nan_to_num(Bk, 0, 0, 0)          # what is left out adds nothing, whatever it holds
    piece = 0.0 if dtype == torch.float32 else 2.0 ** -16                          # two bf16 pieces of dz, 8 bits each
    dz, e = ref["dz"], bounds["dz"] + piece * ref["dz"].abs() + (0 if piece == 0 else 1e-38)
    for name, got, want, err, n in (("features", gf, scale * dz @ Bc, size * (e + (V + 4) * U * dz.abs()) @ Bc.abs(), V),
                                    ("bank", gb, scale * dz.T @ Fc, size * (e + (S + 4) * U * dz.abs()).T @ Fc.abs(), S)):
        within(got, want, torch.nan_to_num(err + half_step(dtype) * (want.abs() + err) + tiny(dtype)), f"gradient of {name}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["none", "bank", "rows"])
@pytest.mark.parametrize("S,V,ch", [(1, 1, 1), (1, 1118, 128), (3, 40, 24), (33, 31, 16), (65, 130, 100), (128, 64, 32), (130, 1000, 64), (257, 70, 129),
                                    (50, 333, 256), (1, 9000, 16), (9000, 3, 16), (300, 1118, 128)])
def test_bank_log_probs_sizes(gpu, S, V, ch, kind, dtype):
    bank_case(gpu, S, V, ch, TYPES[dtype], kind, 0)
    bank_case(gpu, S, V, ch, TYPES[dtype], kind, (1, 5, 16)[S % 3], seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["logp", "entropy", "lse"])
def test_bank_log_probs_single_gradients(gpu, which):
    bank_case(gpu, 70, 200, 32, torch.float32, "rows", 0, which=which)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [-4.0, 0.0, 1e-35, 60.0])
@pytest.mark.parametrize("kind", ["none", "rows"])
def test_bank_log_probs_scales(gpu, kind, scale, dtype):
    bank_case(gpu, 150, 333, 64, TYPES[dtype], kind, 0 if scale == 1e-35 else 5, scale=scale)
    bank_case(gpu, 150, 333, 64, TYPES[dtype], kind, 0, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [300.0, -300.0])
def test_bank_log_probs_scores_far_below_zero(gpu, scale, dtype):
    """The zeros behind the last bank row, and behind the last feature row, must not count beside scores of -300."""
    gen = torch.Generator(device=gpu).manual_seed(3)
    u = torch.nn.functional.normalize(torch.randn(1, 100, generator=gen, device=gpu), dim=1)
    near = lambda n: torch.nn.functional.normalize(u + 0.02 * torch.randn(n, 100, generator=gen, device=gpu), dim=1)
    f, b = near(70).to(TYPES[dtype]), (near(333) * (-1.0 if scale > 0 else 1.0)).to(TYPES[dtype])
    for kind in ("none", "rows"):
        bank_case(gpu, 70, 333, 100, TYPES[dtype], kind, 0, scale=scale, features=f, bank=b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["none", "rows"])
@pytest.mark.parametrize("S,V,ch", [(45000, 3, 16), (3000, 300, 40), (1500, 140, 256)])
def test_bank_log_probs_many_rows_of_few_targets(gpu, S, V, ch, kind, dtype):
    """More rows of one target than one look of a workgroup finds, numbers that are no multiple of a tile, and rows without a target."""
    gen = torch.Generator(device=gpu).manual_seed(S)
    t = torch.randint(-1, 3, (S,), generator=gen, device=gpu)
    bank_case(gpu, S, V, ch, TYPES[dtype], kind, 0, targets=t)


@pytest.mark.gpu
def test_bank_log_probs_far_apart_magnitudes_and_repeated_targets(gpu):
    """f32 rows as pieces: powers of two of the rows change no bit.  All slots share two targets."""
    import nemo_amd
    gen = torch.Generator(device=gpu).manual_seed(8)
    f, b = torch.randn(100, 40, generator=gen, device=gpu), torch.randn(77, 40, generator=gen, device=gpu)
    t = 13 * torch.randint(0, 2, (100,), generator=gen, device=gpu)
    bank_case(gpu, 100, 77, 40, torch.float32, "none", 0, scale=0.5, features=f, bank=b, targets=t)
    p, q = nemo_amd.bank_log_probs(f, b, t, scale=0.5, top=3), nemo_amd.bank_log_probs(f * 2.0 ** 60, b * 2.0 ** -60, t, scale=0.5, top=3)
    assert all(torch.equal(x, y) for x, y in zip(p, q))
    f[3, 0] = INF                                                      # counts: the row is NaN, no other
    r = nemo_amd.bank_log_probs(f, b, t, scale=0.5, top=3)
    assert bool(torch.isnan(r.lse[3])) and int(r.top_index[3, 0]) == -1
    keep = torch.arange(100, device=gpu) != 3
    assert all(torch.equal(x[keep], y[keep]) for x, y in zip(p, r))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bank_log_probs_non_finite_rows_left_out(gpu, dtype):
    """Infinities and NaN in bank rows that are left out for all slots, and in slots for which nothing is left, change nothing."""
    dt = TYPES[dtype]
    gen = torch.Generator(device=gpu).manual_seed(6)
    f = torch.nn.functional.normalize(torch.randn(140, 64, generator=gen, device=gpu), dim=1).to(dt)
    b = torch.nn.functional.normalize(torch.randn(90, 64, generator=gen, device=gpu), dim=1).to(dt)
    w = torch.zeros(140, 90, device=gpu)
    b[7, 3], b[80], b[89, 63] = INF, float("nan"), -INF
    w[:, [7, 80, 89]] = INF
    f[2], f[139, 5] = float("nan"), INF
    w[[2, 139]] = INF
    t = torch.randint(10, 70, (140,), generator=gen, device=gpu)
    t[5], t[6] = 7, -1                                                 # a target that is left out; none
    bank_case(gpu, 140, 90, 64, dt, "rows", 0, features=f, bank=b, weights=w, targets=t)


@pytest.mark.gpu
def test_bank_log_probs_nan_that_counts_and_targets_outside(gpu):
    gen = torch.Generator(device=gpu).manual_seed(6)
    f = torch.nn.functional.normalize(torch.randn(40, 32, generator=gen, device=gpu), dim=1)
    b = torch.nn.functional.normalize(torch.randn(70, 32, generator=gen, device=gpu), dim=1)
    t = torch.randint(0, 70, (40,), generator=gen, device=gpu)
    f[3, 1] = float("nan")
    t[8] = 70
    import nemo_amd
    fl, bl = f.requires_grad_(), b.requires_grad_()
    r = nemo_amd.bank_log_probs(fl, bl, t, top=2)
    bad = torch.zeros(40, dtype=torch.bool, device=gpu)
    bad[3] = True
    assert torch.equal(torch.isnan(r.lse), bad) and torch.equal(torch.isnan(r.entropy), bad) and torch.equal((r.top_index < 0).all(1), bad)
    bad[8] = True
    assert torch.equal(torch.isnan(r.logp), bad)
    gf, gb = torch.autograd.grad(r.logp, (fl, bl), torch.ones(40, device=gpu))
    assert torch.equal(torch.isnan(gf).all(1), bad) and torch.equal(torch.isnan(gf).any(1), bad) and bool(torch.isnan(gb).all())


@pytest.mark.gpu
def test_bank_log_probs_strides_and_starts(gpu):
    import nemo_amd
    gen = torch.Generator(device=gpu).manual_seed(4)
    t = torch.randint(0, 111, (60,), generator=gen, device=gpu)
    for dt in (torch.float32, torch.bfloat16):
        wf, wb = torch.randn(60, 300, generator=gen, device=gpu).to(dt), torch.randn(111, 290, generator=gen, device=gpu).to(dt)
        for off in (0, 1, 8):
            f, b = wf[:, off:off + 64].detach().requires_grad_(), wb[:, 2 * off:2 * off + 64].detach().requires_grad_()
            fc, bc = f.detach().contiguous().requires_grad_(), b.detach().contiguous().requires_grad_()
            r, q = nemo_amd.bank_log_probs(f, b, t, top=3), nemo_amd.bank_log_probs(fc, bc, t, top=3)
            assert all(torch.equal(x, y) for x, y in zip(r, q))
            for x, y in zip(torch.autograd.grad(r.logp.sum(), (f, b)), torch.autograd.grad(q.logp.sum(), (fc, bc))):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_bank_log_probs_gradient_against_differences(gpu):
    """L = sum of logp + 0.5 entropy along a direction.  The values are off by their bounds (64-bit reference), the quotient by their sum / h; the
    third derivative of a log-sum-exp along a direction is at most 2 max|dz|^3 a row, of the entropy 12 max|dz|^3 (1 + max|z|)."""
    import nemo_amd
    S, V, ch, scale, h = 40, 90, 32, 2.0, 0.02
    gen = torch.Generator(device=gpu).manual_seed(8)
    unit = lambda *s: torch.nn.functional.normalize(torch.randn(*s, generator=gen, device=gpu), dim=1)
    f, b, vf, vb = unit(S, ch), unit(V, ch), 0.5 * unit(S, ch), 0.5 * unit(V, ch)
    t = torch.randint(0, V, (S,), generator=gen, device=gpu)

    def value(ff, bb):
        r = nemo_amd.bank_log_probs(ff, bb, t, scale=scale)
        return r.logp.double().sum() + 0.5 * r.entropy.double().sum()
    fl, bl = f.clone().requires_grad_(), b.clone().requires_grad_()
    r = nemo_amd.bank_log_probs(fl, bl, t, scale=scale)
    gf, gb = torch.autograd.grad((r.logp, r.entropy), (fl, bl), (torch.ones(S, device=gpu), torch.full((S,), 0.5, device=gpu)))
    slope = float((gf.double() * vf).sum() + (gb.double() * vb).sum())
    diff = float(value(f + h * vf, b + h * vb) - value(f - h * vf, b - h * vb)) / (2 * h)
    z = scale * f.double() @ b.double().T
    ref = probs_reference(z, t, 0, (None, None, None))
    bounds = probs_bounds(ref, z, torch.full((S,), (ch + 6) * U * scale, device=gpu, dtype=torch.float64), V)
    noise = float((bounds["logp"] + 0.5 * bounds["entropy"]).sum())
    # dz <= scale (|vf| |b| + |f| |vb| + h |vf| |vb|) <= 1.01 scale; z'' = 2 scale <vf, vb> <= scale / 2 enters with first and second derivatives
    dz, zz = 1.01 * scale, 0.5 * scale
    third = S * (2 * dz ** 3 + 3 * dz * zz + 0.5 * (12 * dz ** 3 * (1 + scale) + 12 * dz * zz * (1 + scale)))
    lim = noise / h + h * h / 6 * third
    assert abs(diff - slope) <= lim and lim < 1.0


# ---- together ---------------------------------------------------------------------------------------------------------
def loss_case(dev, multi):
    """A training step's loss as FeatureBankNeMo and MaskCreater give it."""
    from nemo_amd.feature_banks import FeatureBankNeMo, MaskCreater
    torch.manual_seed(1)
    mesh_n, ch, noise, B = [37, 50], 32, 3, 4
    bank = FeatureBankNeMo(input_size=ch, num_pos=sum(mesh_n), num_noise=noise, max_groups=6, momentum=0.9, mesh_n_list=mesh_n).cuda()
    labels = torch.tensor([[0], [1], [0], [1]], dtype=torch.int32, device=dev)
    K = max(mesh_n)
    x = torch.nn.functional.normalize(torch.randn(B, K + noise, ch), dim=2).to(dev)
    visible = (torch.rand(B, K) > 0.3).to(dev)
    for i, l in enumerate([0, 1, 0, 1]):
        visible[i, mesh_n[l]:] = False
    maker = MaskCreater(dist_thr=0.5, kappas={"pos": 0, "near": 1e5, "clutter": 5, "class": 1e5 if multi else 2}, n_noise=noise * 6,
                        verts_ori=[torch.rand(n, 3) for n in mesh_n], device=dev)
    weights, rows = maker(sample_indexs=labels, K_padded=K, vis_mask=visible)
    return bank, x, visible, labels, weights, rows


@pytest.mark.gpu
@pytest.mark.parametrize("multi", [False, True])
def test_bank_loss_of_a_training_step(gpu, multi):
    """The loss of a training step and its gradient with respect to the slots: in one call, through the logits, and in torch in 64 bits."""
    import nemo_amd
    bank, x, visible, labels, weights, rows = loss_case(gpu, multi)
    T = 0.07
    x = x.requires_grad_()
    slots = x[:, :visible.shape[1]][visible]
    memory = bank.memory.clone()
    fused = bank.log_probs(slots, rows, weights, T, top=5)
    loss = -fused.logp.mean()
    (gx,) = torch.autograd.grad(loss, x, retain_graph=True)
    logits = bank.logits(slots, weights, T)
    steps = nemo_amd.log_probs(logits, rows, top=5)
    (gs,) = torch.autograd.grad(-steps.logp.mean(), x, retain_graph=True)
    x64 = x.detach().double().requires_grad_()
    s64 = x64[:, :visible.shape[1]][visible]
    z64 = s64 @ memory.double().T / T - weights.double()
    want = torch.nn.functional.cross_entropy(z64, rows)
    (g64,) = torch.autograd.grad(want, x64)
    # scores up to 1 / T = 14.3 from sums of 32 products, off by (32 + 6) u / T = 3.2e-5 at most, doubled in the probabilities; `logits` has
    # them rounded in f32 as well; a gradient entry is a sum of probabilities times (unit) bank rows / T, divided by the number of slots
    err = 2 * (32 + 8) * U / T + 60 * U
    assert abs(float(loss) - float(want)) <= 2 * err and abs(float(-steps.logp.mean()) - float(want)) <= 2 * err
    bound = 8 * err / T / slots.shape[0]
    within(gx, g64, bound, "gradient, in one call")
    within(gs, g64, bound, "gradient, through the logits")
    for i in range(slots.shape[0]):                                    # the best alternatives are places of the largest scores
        v = z64.detach()[i][fused.top_index[i]]
        assert bool((v >= torch.sort(z64.detach()[i], descending=True).values[:5] - 4 * err).all())
    # forward still returns the similarities and updates the bank
    sim, noise_sim = bank(x, visible, object_labels=labels, vis_mask=visible)
    assert torch.equal(sim, slots @ memory.T) and noise_sim.shape == (4, 3, 87)


@pytest.mark.gpu
def test_bank_loss_other_types_and_widths(gpu):
    """More than 256 channels and half precision go through the logits."""
    from nemo_amd.feature_banks import FeatureBankNeMo
    torch.manual_seed(2)
    for ch, dt in ((300, torch.float32), (64, torch.float16), (64, torch.bfloat16)):
        bank = FeatureBankNeMo(input_size=ch, num_pos=60, num_noise=0).cuda()
        f = torch.nn.functional.normalize(torch.randn(20, ch), dim=1).to(gpu).to(dt)
        rows = torch.randint(0, 60, (20,), device=gpu)
        r = bank.log_probs(f, rows, T=0.5, top=1)
        z = 2.0 * f.double() @ bank.memory.to(dt).double().T
        want = torch.log_softmax(z, 1).gather(1, rows[:, None])[:, 0]
        err = 2 * ((ch + 6) * U * 2 * float(bank.memory.norm(dim=1).max()) + 60 * U)
        if dt == torch.float16:
            err += 2 * half_step(dt) * float(z.abs().max())            # the logits are rounded to their type
        within(r.logp, want, err, "logp")


@pytest.mark.gpu
def test_results_repeat(gpu):
    import nemo_amd
    gen = torch.Generator(device=gpu).manual_seed(0)
    x, w = torch.randn(700, 96, generator=gen, device=gpu).requires_grad_(), torch.randn(40, 96, generator=gen, device=gpu).requires_grad_()
    t = torch.randint(0, 40, (700,), generator=gen, device=gpu)

    def all_of():
        y = nemo_amd.linear(x, w, activation="gelu")
        r, s = nemo_amd.log_probs(y, t, top=4), nemo_amd.bank_log_probs(x, w, t, top=4)
        return [y, *r, *s, *torch.autograd.grad(r.logp.sum() + s.entropy.sum() + s.logp.sum(), (x, w))]
    first = all_of()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, all_of()))


@pytest.mark.gpu
def test_other_stream_and_captured_graph(gpu):
    """On a side stream, and captured with its backward pass: every replay equals the eager result, with eager work in between."""
    import nemo_amd
    gen = torch.Generator(device=gpu).manual_seed(0)
    S, V, ch = 200, 333, 64
    unit = lambda n: torch.nn.functional.normalize(torch.randn(n, ch, generator=gen, device=gpu), dim=1)
    x, w, b = unit(S).requires_grad_(), (0.1 * torch.randn(ch, ch, generator=gen, device=gpu)).requires_grad_(), torch.zeros(ch, device=gpu).requires_grad_()
    bank, t = unit(V).requires_grad_(), torch.randint(0, V, (S,), generator=gen, device=gpu)
    weights = torch.rand(S, V, generator=gen, device=gpu)

    def step():
        f = nemo_amd.linear(x, w, b, residual=x, activation="silu")
        r = nemo_amd.bank_log_probs(f, bank, t, weights, scale=5.0, top=3)
        q = nemo_amd.log_probs(nemo_amd.linear(f, bank), t, weights)
        loss = -(r.logp + q.logp + 0.1 * r.entropy).mean()
        return [loss, r.logp, r.top_index, *torch.autograd.grad(loss, (x, w, b, bank))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [o.detach().clone() for o in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(on_side, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(unit(S))
            bank.copy_(unit(V))
            t.copy_(torch.randint(0, V, (S,), generator=gen, device=gpu))
        graph.replay()
        got = [o.detach().clone() for o in out]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, step())), f"replay {i}"


@pytest.mark.gpu
def test_two_graphs_and_calls_without_gradients(gpu):
    """Two captured graphs replayed in turn, each with its own workspace; results without gradients are those with them."""
    import nemo_amd
    gen = torch.Generator(device=gpu).manual_seed(1)
    data = [(torch.randn(S, 48, generator=gen, device=gpu).requires_grad_(), torch.randn(V, 48, generator=gen, device=gpu).requires_grad_(),
             torch.randint(0, V, (S,), generator=gen, device=gpu)) for S, V in ((70, 301), (500, 90))]

    def step(x, bank, t):
        y = nemo_amd.linear(x, bank, alpha=0.1)
        r, q = nemo_amd.bank_log_probs(x, bank, t, scale=0.1, top=2), nemo_amd.log_probs(y, t, top=2)
        return [*r, *q, *torch.autograd.grad((r.logp + q.entropy).sum(), (x, bank))]
    eager = [[o.detach().clone() for o in step(*d)] for d in data]
    with torch.no_grad():
        for (x, bank, t), e in zip(data, eager):
            free = [*nemo_amd.bank_log_probs(x, bank, t, scale=0.1, top=2), *nemo_amd.log_probs(nemo_amd.linear(x, bank, alpha=0.1), t, top=2)]
            assert not any(o.requires_grad for o in free) and all(torch.equal(p, q) for p, q in zip(free, e))
    graphs = []
    for d in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*d)
        graphs.append((graph, out))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), e in zip(graphs, eager):
            assert all(torch.equal(p.detach(), q) for p, q in zip(out, e))


# ---- the C entries' refusals (no launch happens: run on the CPU) ----------------------------------------------------------
def _lib_or_skip():
    import os
    from nemo_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libnemo_hip.so is not built")
    return _lib.load()


def test_entry_refusals():
    lib = _lib_or_skip()
    p = C.c_void_p(4096)                                               # never read: every call below is refused or empty
    err = lambda: lib.nemo_last_error().decode()

    def linear(M=4, N=4, K=8, dt=0, act=0, x=p, w=p, y=p, ldx=8, ldw=8, r=None, ldr=4, ws=None, nbytes=0):
        return lib.nemo_linear(x, ldx, w, ldw, None, r, ldr, M, N, K, dt, act, 1.0, 1.0, y, None, ws, nbytes, None)
    assert linear(M=-1) == -1 and linear(dt=7) == -1 and linear(act=9) == -1 and linear(x=None) == -1 and linear(y=None) == -1
    assert linear(ldx=7) == -1 and "stride" in err()
    assert linear(r=p, ldr=3) == -1 and linear(M=1 << 33) == -2 and linear(M=1 << 20, N=1 << 20) == -2 and "too large" in err()
    assert linear(K=7, ldx=7, ldw=7) == -1 and "workspace" in err()     # rows off 16 bytes need their copies
    assert linear(M=0) == 0 and linear(N=0) == 0

    def linear_bwd(M=4, N=4, K=8, g=p, x=p, w=p, pre=None, act=0, gx=p, gw=p):
        return lib.nemo_linear_backward(g, N, x, K, w, K, pre, M, N, K, 0, act, 1.0, 1.0, gx, gw, None, None, None, 0, None)
    assert linear_bwd(g=None) == -1 and linear_bwd(x=None) == -1 and linear_bwd(w=None) == -1 and linear_bwd(act=2) == -1 and "pre" in err()

    def probs(S=4, V=9, dt=0, top=0, x=p, t=p, ld=9, w=None, ldw=0, stats=None, ws=None, nbytes=0):
        return lib.nemo_log_probs(x, ld, w, ldw, t, S, V, dt, 1.0, top, None, None, None, stats, None, None, ws, nbytes, None)
    assert probs(S=-1) == -1 and probs(dt=3) == -1 and probs(top=17) == -2 and probs(top=2) == -1 and probs(x=None) == -1 and probs(t=None) == -1
    assert probs(ld=8) == -1 and probs(w=p, ldw=5) == -1 and probs(S=1 << 24) == -2 and probs(V=1 << 31, ld=1 << 31) == -2
    assert probs(S=1, V=1 << 20, ld=1 << 20) == -1 and "workspace" in err()
    assert probs(stats=C.c_void_p(4100)) == -1 and probs(S=0) == 0
    assert lib.nemo_log_probs_backward(p, 9, None, 0, p, None, None, None, None, 4, 9, 0, 1.0, p, None) == -1
    assert lib.nemo_log_probs_backward(p, 8, None, 0, p, p, None, None, None, 4, 9, 0, 1.0, p, None) == -1

    def bank(S=4, V=9, ch=16, dt=0, top=0, f=p, b=p, t=p, ldf=16, ldb=16, ws=None, nbytes=0):
        return lib.nemo_bank_log_probs(f, ldf, b, ldb, None, 0, t, S, V, ch, dt, 1.0, top, None, None, None, None, None, None, ws, nbytes, None)
    assert bank(S=-1) == -1 and bank(ch=0) == -1 and bank(ch=257, ldf=257, ldb=257) == -2 and bank(dt=2) == -2 and bank(top=17) == -2
    assert bank(f=None) == -1 and bank(t=None) == -1 and bank(ldf=15) == -1 and bank(S=1 << 24) == -2 and bank(S=0) == 0
    assert bank() == -1 and "workspace" in err()
    assert lib.nemo_bank_log_probs_backward(p, 16, p, 16, None, 0, p, None, None, None, None, 4, 9, 16, 0, 1.0, 0, p, p, None, 0, None) == -1
    assert lib.nemo_bank_log_probs_backward(p, 16, p, 16, None, 0, p, p, None, None, None, 4, 9, 16, 0, 1.0, 0, p, p, None, 0, None) == -1
    assert lib.nemo_linear_workspace(p, 8, p, 8, 4, 4, 8, 0) == 0       # aligned rows and enough tiles' worth of nothing to split


def test_entry_refuses_strides():
    lib = _lib_or_skip()
    p = C.c_void_p(4096)
    assert lib.nemo_linear(p, 1 << 21, p, 8, None, None, 0, 4, 4, 8, 0, 0, 1.0, 1.0, p, None, None, 0, None) == -2
    assert "4 MiB" in lib.nemo_last_error().decode()
    assert lib.nemo_bank_log_probs_backward(p, 16, p, 16, p, 1 << 28, p, p, None, None, None, 4, 9, 16, 0, 1.0, 0, p, p, p, 1 << 30, None) == -2
    assert "2^27" in lib.nemo_last_error().decode()


def test_host_tensors_are_refused():
    import nemo_amd
    x, t = torch.zeros(4, 16), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: nemo_amd.linear(x, x), lambda: nemo_amd.log_probs(x, t), lambda: nemo_amd.bank_log_probs(x, x, t)):
        with pytest.raises(RuntimeError, match="CPU"):
            call()
    for call in (lambda: nemo_amd.linear(None, x), lambda: nemo_amd.linear([1.0], x), lambda: nemo_amd.log_probs(None, t),
                 lambda: nemo_amd.bank_log_probs(None, x, t)):
        with pytest.raises(TypeError):
            call()
