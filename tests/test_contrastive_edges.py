"""The contrastive loss's operators where sizes, values and strides leave the ordinary range; tolerances as in test_contrastive.py."""
import ctypes as C

import pytest
import torch

from tests.test_contrastive import ACT, CURVE, INF, TYPES, U, bank_case, half_step, loss_case, tiny, within


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [300.0, -300.0])
@pytest.mark.parametrize("S,V,ch", [(70, 333, 100), (33, 31, 24), (140, 65, 200)])
def test_scores_far_below_zero_with_a_list(gpu, S, V, ch, scale, dtype):
    """The zeros behind the last bank row must not count beside scores of -300, in the forms for lists too.  Rows on a grid of 1/128: products are
    exact, and so is their multiple by 300, so the order of the best entries is that of 64 bits."""
    gen = torch.Generator(device=gpu).manual_seed(3)
    u = torch.nn.functional.normalize(torch.randn(1, ch, generator=gen, device=gpu), dim=1)
    near = lambda n: torch.round(128 * torch.nn.functional.normalize(u + 0.02 * torch.randn(n, ch, generator=gen, device=gpu), dim=1)) / 128
    f, b = near(S).to(TYPES[dtype]), (near(V) * (-1.0 if scale > 0 else 1.0)).to(TYPES[dtype])
    for top in (1, 5, 16):
        bank_case(gpu, S, V, ch, TYPES[dtype], "none", top, scale=scale, features=f, bank=b)
    bank_case(gpu, S, V, ch, TYPES[dtype], "rows", 5, scale=scale, features=f, bank=b)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_linear_pre_activations_beyond_f16(gpu, act):
    """Half of the pre-activations lie beyond the largest f16, where the slopes are 0 and 1 (to far more than 64 bits); the results on the negative side
    are the residual, and every gradient is what 64 bits give.  The others are ordinary: their slopes are off by the rounding of the kept
    pre-activation (half a step) times the curvature."""
    import nemo_amd
    M, N, K, dt = 50, 36, 8, torch.float16
    gen = torch.Generator(device=gpu).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=gpu)
    x, w = rnd(M, K), rnd(N, K) * K ** -0.5
    x[:, 0], w[:, 0] = 0, 0
    x[:, 0] = torch.where(torch.arange(M, device=gpu) % 2 == 0, 300.0, -240.0)
    w[::2, 0] = 280.0                                                  # 84000 and -67200
    x, w, r, g = (t.to(dt) for t in (x, w, rnd(M, N), rnd(M, N)))
    leaves = [t.clone().requires_grad_() for t in (x, w, torch.zeros(N, device=gpu, dtype=dt), r)]
    y = nemo_amd.linear(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, g)
    X, W, G, uT = x.double(), w.double(), g.double(), half_step(dt)
    z = (X @ W.T).requires_grad_()
    (slope,) = torch.autograd.grad(ACT[act](z).sum(), z)
    z = z.detach()
    far = z.abs() > 1000
    assert bool((z.abs()[far] > 65520).all()) and int(far.sum()) == M * N // 2 and bool((far & (z < 0)).any())
    assert torch.equal(y.detach()[far & (z < 0)], r[far & (z < 0)]) and bool((y[far & (z > 0)] == INF).all())
    z_err = (K + 4) * U * (X.abs() @ W.abs().T)
    s_err = CURVE[act] * (z_err + uT * z.abs() + tiny(dt)) + 16 * U * (1 + z.abs())
    if act == "relu":
        s_err = (z.abs() <= z_err).double()
    s_err = torch.where(far, torch.zeros_like(z), s_err)
    dz, e = G * slope, G.abs() * s_err
    dz_err = e + uT * (dz.abs() + e) + tiny(dt)                        # dz is rounded in front of the two products
    want = (dz @ W, dz.T @ X, dz.sum(0), G)
    err = (dz_err @ W.abs() + (N + 4) * U * (dz.abs() + dz_err) @ W.abs(), dz_err.T @ X.abs() + (M + 4) * U * (dz.abs() + dz_err).T @ X.abs(),
           e.sum(0) + (M + 4) * U * (dz.abs() + e).sum(0), torch.zeros_like(G))
    for name, got, v, b in zip(("x", "weight", "bias", "residual"), grads, want, err):
        assert bool(torch.isfinite(got).all()), name
        within(got, v, b + uT * (v.abs() + b) + tiny(dt), f"gradient of {name}")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_linear_pre_activation_that_rounds_to_infinity_in_bf16(gpu, act):
    """-1.998 2^127 is a number in f32 and rounds to -infinity in bf16: the slope there is 0."""
    import nemo_amd
    x = torch.full((1, 2), -2.0 ** 64, device=gpu, dtype=torch.bfloat16).requires_grad_()
    w = torch.tensor([[1.9921875 * 2.0 ** 63, 0.005859375 * 2.0 ** 63]], device=gpu, dtype=torch.bfloat16).requires_grad_()
    y = nemo_amd.linear(x, w, activation=act)
    gx, gw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert not y.any() and not gx.any() and not gw.any()


@pytest.mark.gpu
def test_forward_mode_is_refused(gpu):
    """No tangent is computed: a dual tensor is refused instead of being taken for a constant, with and without gradients."""
    import nemo_amd
    from torch.autograd import forward_ad
    x, w, t = torch.ones(4, 16, device=gpu), torch.ones(9, 16, device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu)
    weights = torch.zeros(9, device=gpu)
    bank_logits = lambda v: nemo_amd.linear(v, w)
    calls = (bank_logits, lambda v: nemo_amd.linear(x, w, residual=torch.ones(4, 9, device=gpu), bias=v[0, :9]), lambda v: nemo_amd.log_probs(v, t),
             lambda v: nemo_amd.bank_log_probs(v, w, t), lambda v: nemo_amd.log_probs(x, t, weights=v[0]))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward"):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
                call(dual)
        assert torch.equal(nemo_amd.linear(x, w), torch.full((4, 9), 16.0, device=gpu))       # ordinary tensors are taken
        assert not nemo_amd.log_probs(x, t, weights=torch.zeros(16, device=gpu)).logp.isnan().any()
    with pytest.raises(RuntimeError):
        torch.func.jvp(bank_logits, (x,), (x,))
    leaf = x.clone().requires_grad_()                                  # a backward pass of a dual gradient
    for y in (nemo_amd.linear(leaf, w), nemo_amd.log_probs(leaf, t).lse, nemo_amd.bank_log_probs(leaf, w, t).lse):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward"):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.gpu
def test_linear_rows_of_results_beyond_the_backward_pass(gpu):
    """Results of more than 4 MiB a row: taken without gradients of x and weight, refused with them before anything runs."""
    import nemo_amd
    N = (1 << 20) + 8
    x, w, b = torch.ones(2, 4, device=gpu), torch.ones(N, 4, device=gpu), torch.zeros(N, device=gpu)
    assert bool((nemo_amd.linear(x, w, b) == 4.0).all())
    for leaf in (x, w):
        leaf.requires_grad_()
        with pytest.raises(ValueError, match="4 MiB"):
            nemo_amd.linear(x, w, b)
        leaf.requires_grad_(False)
    y = nemo_amd.linear(x, w, b.requires_grad_())
    (gb,) = torch.autograd.grad(y, b, torch.ones_like(y))
    assert bool((gb == 2.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_gradient_with_rows_far_apart(gpu, dtype):
    """An incoming gradient that is a slice of rows more than 4 MiB long."""
    import nemo_amd
    dt = TYPES[dtype]
    gen = torch.Generator(device=gpu).manual_seed(2)
    x, w = (torch.randn(n, 40, generator=gen, device=gpu).to(dt).requires_grad_() for n in (5, 64))
    wide = torch.randn(5, (1 << 21) + 64, generator=gen, device=gpu).to(dt)
    y = nemo_amd.linear(x, w)
    for g in (wide[:, :64], wide[:, 1:65]):
        got = torch.autograd.grad(y, (x, w), g, retain_graph=True)
        want = torch.autograd.grad(y, (x, w), g.contiguous(), retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_entry_takes_gradients_with_rows_far_apart():
    """The C entry asks for a copy of such rows instead of refusing them; a row itself may be no longer than 4 MiB."""
    from tests.test_contrastive import _lib_or_skip
    lib = _lib_or_skip()
    p = C.c_void_p(4096)
    near, far = (lib.nemo_linear_backward_workspace(p, ld, p, 8, p, 8, 4, 8, 8, 0, 0) for ld in (8, (1 << 20) + 4))
    assert far == near + 256                                           # 4 rows of 32 bytes, in whole 256s

    def backward(ldg, N):
        return lib.nemo_linear_backward(p, ldg, p, 8, p, 8, None, 4, N, 8, 0, 0, 1.0, 1.0, p, p, None, None, None, 0, None)
    assert backward((1 << 20) + 4, 8) == -1 and "workspace" in lib.nemo_last_error().decode()
    assert backward((1 << 20) + 4, (1 << 20) + 4) == -2 and "4 MiB" in lib.nemo_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bank_weights_with_rows_far_apart(gpu, dtype):
    """Rows of weights more than 2^27 elements apart, forward and backward."""
    import nemo_amd
    gen = torch.Generator(device=gpu).manual_seed(2)
    f, b = (torch.randn(n, 32, generator=gen, device=gpu).to(TYPES[dtype]).requires_grad_() for n in (3, 70))
    t = torch.tensor([0, 69, -1], device=gpu)
    far = torch.zeros(2 * ((1 << 27) + 8) + 70, device=gpu).as_strided((3, 70), ((1 << 27) + 8, 1))
    far.copy_(torch.rand(3, 70, generator=gen, device=gpu))
    out = []
    for weights in (far, far.contiguous()):
        r = nemo_amd.bank_log_probs(f, b, t, weights, scale=0.2, top=2)
        out.append([*r, *torch.autograd.grad((r.logp + r.entropy).sum(), (f, b))])
    assert all(torch.equal(p, q) for p, q in zip(*out))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_operands_with_rows_far_apart(gpu, dtype):
    """Slices of rows more than 4 MiB long, on 16 bytes and off them."""
    import nemo_amd
    dt = TYPES[dtype]
    gen = torch.Generator(device=gpu).manual_seed(2)
    wide = torch.randn(5, (1 << 21) + 64, generator=gen, device=gpu).to(dt)
    for x, w in ((wide[:, :40], wide[:3, 64:104]), (wide[:, 1:41], wide[:3, 3:43])):
        out = []
        for leaves in ([x.detach().requires_grad_(), w.detach().requires_grad_()], [t.contiguous().requires_grad_() for t in (x, w)]):
            y = nemo_amd.linear(*leaves, activation="silu")
            out.append([y, *torch.autograd.grad(y.sum(), leaves)])
        assert all(torch.equal(p, q) for p, q in zip(*out))


@pytest.mark.gpu
def test_host_targets_in_a_capture(gpu):
    """Targets on the host are copied with a blocking copy, which a capture does not take: refused, and the capture goes on."""
    import nemo_amd
    x, w, t = torch.randn(4, 16, device=gpu), torch.randn(9, 16, device=gpu), torch.zeros(4, dtype=torch.int64)
    eager = nemo_amd.log_probs(x, t).lse
    assert torch.equal(eager, nemo_amd.log_probs(x, t.to(gpu)).lse)
    t_dev = t.to(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: nemo_amd.log_probs(x, t), lambda: nemo_amd.bank_log_probs(x, w, t)):
            with pytest.raises(RuntimeError, match="on the host"):
                call()
        lse = nemo_amd.log_probs(x, t_dev).lse
    for _ in range(3):
        lse.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(lse, eager)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_bank_logits_take_the_weights_of_log_probs(gpu, dtype):
    """MaskCreater's f32 weights with slots of any type.  They are rounded to the slots' type (a weight beyond f16 leaves its place out), the result
    once more."""
    dt = TYPES[dtype]
    bank, x, visible, _, weights, rows = loss_case(gpu, True)
    slots = x[:, :visible.shape[1]][visible].to(dt)
    weights = weights + 0.3 * (torch.arange(weights.shape[1], device=gpu) % 3)
    T = 0.07
    leaf = weights.clone().requires_grad_()
    got = bank.logits(slots, leaf, T)
    assert got.dtype == dt
    w = weights.to(dt).double()
    S, B = slots.double(), bank.memory.to(dt).double()
    want = S @ B.T / T - w
    err = 2 * (32 + 8) * U / T * (S.abs() @ B.abs().T) + 4 * U * want.abs()
    want_t = torch.where(want.abs() > torch.finfo(dt).max, torch.sign(want) * INF, want)
    within(got, want_t, torch.nan_to_num(err + half_step(dt) * (want.abs() + err), 0, 0, 0), "logits")
    (gw,) = torch.autograd.grad(got, leaf, torch.ones_like(got))
    assert gw.dtype == torch.float32 and bool((gw == -1.0).all())
    assert torch.equal(bank.logits(slots, weights.to(dt), T), got.detach())
    assert torch.equal(bank.logits(slots, weights[0], T), bank.logits(slots, weights[:1].expand_as(weights), T))
    r = bank.log_probs(slots, rows, weights, T)
    assert bool(torch.isfinite(r.logp).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bank_scale_near_the_largest_number(gpu, dtype):
    """scale log2 e is beyond f32: products of 0 and of 2^-126 give scores of 0 and 3.5."""
    f, b = (torch.eye(n, 64, device=gpu).mul_(2.0 ** -63).to(TYPES[dtype]) for n in (64, 50))
    for scale in (3.0e38, -3.0e38):
        bank_case(gpu, 64, 50, 64, TYPES[dtype], "none", 0, scale=scale, features=f, bank=b)


def test_numbers_beyond_f32_are_refused():
    from nemo_amd import contrastive
    for v in (1e39, -1e39, 3.4028236e38):
        with pytest.raises(ValueError, match="finite"):
            contrastive._number("linear", "alpha", v)
    assert contrastive._number("linear", "alpha", 3.4028234663852886e38) == 3.4028234663852886e38


def test_entries_refuse_workspaces_off_16_bytes():
    from tests.test_contrastive import _lib_or_skip
    lib = _lib_or_skip()
    p, ws, n = C.c_void_p(4096), C.c_void_p(4104), 1 << 30
    for rc in (lib.nemo_linear(p, 7, p, 7, None, None, 0, 4, 4, 7, 0, 0, 1.0, 1.0, p, None, ws, n, None),
               lib.nemo_linear_backward(p, 8, p, 7, p, 7, None, 4, 8, 7, 0, 0, 1.0, 1.0, p, p, None, None, ws, n, None),
               lib.nemo_log_probs(p, 1 << 20, None, 0, p, 1, 1 << 20, 0, 1.0, 0, p, None, None, None, None, None, ws, n, None),
               lib.nemo_bank_log_probs(p, 16, p, 16, None, 0, p, 4, 9, 16, 0, 1.0, 0, p, None, None, None, None, None, ws, n, None),
               lib.nemo_bank_log_probs_backward(p, 16, p, 16, None, 0, p, p, None, None, None, 4, 9, 16, 0, 1.0, 0, p, p, ws, n, None)):
        assert rc == -1 and "16 bytes" in lib.nemo_last_error().decode()
