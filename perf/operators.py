"""The cases on which the operators of the contrastive bank loss are measured: `linear` (matrix product with bias, activation and
residual), `log_probs` (log probabilities, entropy and top alternatives of logits) and `bank_log_probs` (the same straight from
features and bank).  `own` chooses between elementary torch operations in 32 bits and the package's kernels."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- cases ----------------------------------------------------------------------------------------------------------
def _linear(name, dtype, m, n, k, act="none", bias=False, residual=False, alpha=1.0, beta=1.0, train=False):
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "n": n, "k": k, "act": act, "bias": bias, "residual": residual,
            "alpha": alpha, "beta": beta, "train": train}


def _log_probs(name, dtype, rows, cols, scale=1.0, top=0, weights="none", train=False):
    return {"name": name, "op": "log_probs", "dtype": dtype, "rows": rows, "cols": cols, "scale": scale, "top": top,
            "weights": weights, "train": train}


def _bank(name, dtype, rows, cols, channels, scale=16.0, top=0, weights="none", train=False):
    return {"name": name, "op": "bank_log_probs", "dtype": dtype, "rows": rows, "cols": cols, "channels": channels, "scale": scale,
            "top": top, "weights": weights, "train": train}


def listed():
    return [
        # the logits of a few vertex slots against one category's bank (1118 vertices + 512 images x 5 clutter rows), weights subtracted
        _linear("linear_few_slots", "f32", 20, 3678, 128, residual=True, alpha=16.0, beta=-1.0),
        # the logits of five images' vertex slots against a bank of twelve categories with its clutter rows, weights subtracted
        _linear("linear_bank_weights", "f32", 5590, 15976, 128, residual=True, alpha=16.0, beta=-1.0),
        # the 1 x 1 projection of a backbone's last layer on twenty 80 x 100 maps
        _linear("linear_head", "bf16", 160000, 128, 2048, act="relu", bias=True),
        # a wide layer on a long batch: the matrix product itself
        _linear("linear_wide", "bf16", 8192, 4096, 4096, act="gelu", bias=True, residual=True),
        # forward and backward of a layer whose sizes fit no tile and whose rows are not aligned
        _linear("linear_odd_train", "f16", 8191, 1001, 515, act="silu", bias=True, residual=True, train=True),
        # one slot looked up among one category's vertices: launch and latency
        _log_probs("log_probs_one_row", "f32", 1, 1118, scale=2.0, top=5),
        # evaluation: which of twelve categories' vertices every pixel of an 80 x 100 map shows
        _log_probs("log_probs_pixels", "f32", 8000, 13416, scale=2.0, top=5),
        # a training step on logits of a long list of classes, odd in number
        _log_probs("log_probs_train", "bf16", 4096, 100003, train=True),
        # one slot straight from its features
        _bank("bank_one_slot", "f32", 1, 1118, 128, top=1),
        # evaluation of every pixel straight from the feature map
        _bank("bank_pixels", "f32", 8000, 13416, 128, top=5),
        # a training step: the visible slots of a batch of 20 images against one category's bank, weights for every pair
        _bank("bank_weights_train", "f32", 10007, 3678, 128, weights="rows", train=True),
        # a training step on a large batch against the bank of twelve categories with its clutter rows
        _bank("bank_train", "bf16", 32768, 15976, 128, train=True),
    ]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "log_probs", "bank_log_probs"])
    train = rng.random() < 0.5
    if op == "linear":
        dtype = rng.choice(["f32", "bf16", "f16"])
        n, k = _spread(rng, 16, 16384), _spread(rng, 16, 4096)
        if rng.random() < 0.5:                                    # half of the layers have widths of whole 64s
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        limit = 4.0e10 if dtype == "f32" else 2.7e11
        room = limit / ((6.0 if train else 2.0) * n * k)
        m = _spread(rng, 1, int(max(1, min(160000, room, 3.0e8 / max(n, k)))))
        residual = rng.random() < 0.5
        return _linear(None, dtype, m, n, k, act=rng.choice(["none", "relu", "gelu", "silu"]), bias=rng.random() < 0.6, residual=residual,
                       alpha=rng.choice([1.0, 0.5, 16.0 / k]), beta=rng.choice([1.0, -1.0, 0.5]) if residual else 1.0, train=train)
    weights = rng.choice(["none", "none", "bank", "rows"])
    scale = rng.choice([1.0, 4.0, 7.5, 8.0])
    top = 0 if train else rng.choice([0, 1, 5, 8])
    if op == "log_probs":
        dtype = rng.choice(["f32", "bf16", "f16"])
        cols = _spread(rng, 60, 131072)
        rows = _spread(rng, 1, int(max(1, min(32768, 1.0e8 / cols))))
        return _log_probs(None, dtype, rows, cols, scale=rng.choice([1.0, 0.5, 1.5]), top=top, weights=weights, train=train)
    dtype = rng.choice(["f32", "bf16"])
    channels = rng.choice([16, 24, 32, 64, 100, 128, 128, 256])
    cols = _spread(rng, 60, 16000)
    room = 1.2e8 if dtype == "f32" else 4.0e8
    if weights == "rows":
        room = 1.0e8
    rows = _spread(rng, 1, int(max(1, min(32768, room / cols * (128.0 / max(channels, 128))))))
    return _bank(None, dtype, rows, cols, channels, scale=scale, top=top, weights=weights, train=train)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _normal(gen, *shape, dtype=torch.float32, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _weights(gen, kind, rows, cols, targets):
    """Weights as the contrastive loss has them: 0 for most rows of the bank, a constant for its last sixth (clutter), a large
    number around the target (its neighbours on the mesh), +inf for places that are left out."""
    if kind == "none":
        return None
    tail = torch.zeros(cols, device="cuda")
    tail[cols - cols // 6:] = 5.0
    if kind == "bank":
        gone = torch.rand(cols, generator=gen, device="cuda") < 0.05
        gone[0] = False
        return tail.masked_fill(gone, float("inf"))
    w = tail.expand(rows, cols).clone()
    for step in (-2, -1, 1, 2):
        near = (targets.clamp(min=0) + step) % cols
        w[torch.arange(rows, device="cuda"), near] = 1.0e5
    w[:, cols // 2] = float("inf")
    rows_t = torch.arange(rows, device="cuda")
    w[rows_t, targets.clamp(min=0)] = 0.0
    return w


def _unit(t):
    return torch.nn.functional.normalize(t, dim=1)


def _unit_grid(t):
    """Unit vectors on a grid of 1/256, as features kept in 8 bits with a common step are: dot products of them are whole
    multiples of 2^-16, so which rows are the best ones does not hang on the order of a sum."""
    return torch.round(_unit(t) * 256.0) / 256.0


def _targets(gen, rows, cols):
    t = torch.randint(0, cols, (rows,), generator=gen, device="cuda")
    if rows > 16:
        t[torch.rand(rows, generator=gen, device="cuda") < 0.02] = -1                  # slots without a target
    return t


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, train = _TYPES[case["dtype"]], case["train"]
    st = {"case": case}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        st["x"] = _normal(gen, m, k, dtype=dt)
        st["weight"] = _normal(gen, n, k, dtype=dt, std=k ** -0.5)
        st["bias"] = _normal(gen, n, dtype=dt) if case["bias"] else None
        st["residual"] = _normal(gen, m, n, dtype=dt) if case["residual"] else None
        st["grad"] = _normal(gen, m, n, dtype=dt) if train else None
        leaves = ("x", "weight", "bias", "residual")
    else:
        rows, cols = case["rows"], case["cols"]
        st["targets"] = _targets(gen, rows, cols)
        st["weights"] = _weights(gen, case["weights"], rows, cols, st["targets"])
        if case["weights"] == "bank":                              # a slot whose own row is left out has no target
            st["targets"] = torch.where(torch.isinf(st["weights"])[st["targets"].clamp(min=0)], -1, st["targets"])
        if case["op"] == "log_probs":
            logits = _normal(gen, rows, cols, std=2.0)
            if dt == torch.float32:
                logits = torch.round(logits * 4096.0) / 4096.0
            st["logits"] = logits.to(dt)
            leaves = ("logits",)
        else:
            unit = _unit_grid if case["top"] else _unit
            bank = unit(_normal(gen, cols, case["channels"]))
            noise = _normal(gen, rows, case["channels"], std=2.0 * case["channels"] ** -0.5)
            st["features"] = unit(bank[st["targets"].clamp(min=0)] + noise).to(dt)
            st["bank"] = bank.to(dt)
            leaves = ("features", "bank")
        if train:
            # a mean over the rows, some of them weighted down, with a small reward for entropy; in f16 with a loss scale
            share = (1024.0 if dt == torch.float16 else 1.0) / rows
            st["grad_logp"] = -share * torch.rand(rows, generator=gen, device="cuda")
            st["grad_entropy"] = -0.01 * share * torch.rand(rows, generator=gen, device="cuda")
    if train:
        st["leaves"] = [name for name in leaves if st[name] is not None]
        for name in st["leaves"]:
            st[name].requires_grad_(True)
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    import nemo_amd
    case = st["case"]
    if case["op"] == "linear":
        y = nemo_amd.linear(st["x"], st["weight"], bias=st["bias"], residual=st["residual"], activation=case["act"], alpha=case["alpha"],
                            beta=case["beta"])
        if not case["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, [st[name] for name in st["leaves"]], st["grad"])
        return {"y": y.detach(), **{"grad_" + name: g for name, g in zip(st["leaves"], grads)}}
    if case["op"] == "log_probs":
        r = nemo_amd.log_probs(st["logits"], st["targets"], weights=st["weights"], scale=case["scale"], top=case["top"])
    else:
        r = nemo_amd.bank_log_probs(st["features"], st["bank"], st["targets"], weights=st["weights"], scale=case["scale"], top=case["top"])
    out = {"logp": r.logp, "entropy": r.entropy, "lse": r.lse}
    if case["top"]:
        out["top_logp"], out["top_index"] = r.top_logp, r.top_index
    if case["train"]:
        grads = torch.autograd.grad((r.logp, r.entropy), [st[name] for name in st["leaves"]], (st["grad_logp"], st["grad_entropy"]))
        out = {key: v.detach() for key, v in out.items()}
        out.update({"grad_" + name: g for name, g in zip(st["leaves"], grads)})
    return out


def _activate(z, act):
    """-> (act(z), its derivative as a function without arguments)."""
    if act == "none":
        return z, lambda: torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0.0), lambda: (z > 0).to(z.dtype)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, lambda: s * (1.0 + z * (1.0 - s))
    phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * phi, lambda: phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_linear(st):
    case = st["case"]
    dt = st["x"].dtype
    x, w = st["x"].detach().float(), st["weight"].detach().float()
    z = (x @ w.T) * case["alpha"]
    if st["bias"] is not None:
        z = z + st["bias"].detach().float()
    y, slope = _activate(z, case["act"])
    if st["residual"] is not None:
        y = y + case["beta"] * st["residual"].detach().float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = st["grad"].float()
        dz = dy * slope()
        out["grad_x"] = ((dz @ w) * case["alpha"]).to(dt)
        out["grad_weight"] = ((dz.T @ x) * case["alpha"]).to(dt)
        if st["bias"] is not None:
            out["grad_bias"] = dz.sum(dim=0).to(dt)
        if st["residual"] is not None:
            out["grad_residual"] = (case["beta"] * dy).to(dt)
    return out


def _plain_scores(st):
    """-> z [rows, cols] in 32 bits, -inf where a place is left out."""
    case = st["case"]
    if case["op"] == "log_probs":
        z = st["logits"].detach().float() * case["scale"]
    else:
        z = (st["features"].detach().float() @ st["bank"].detach().float().T) * case["scale"]
    if st["weights"] is not None:
        z = torch.where(st["weights"] == float("inf"), torch.full_like(z, -float("inf")), z - st["weights"])
    return z


def _plain_top(z, log_p, k):
    """The k largest of every row, the lowest index first among equals; -1 where nothing is left."""
    rest, places = z.clone(), torch.arange(z.shape[1], device=z.device)
    values, index = [], []
    for _ in range(k):
        best = rest.amax(dim=1, keepdim=True)
        at = torch.where(rest == best, places, z.shape[1]).amin(dim=1, keepdim=True)
        rest.scatter_(1, at, -float("inf"))
        none = best == -float("inf")
        values.append(torch.where(none, best, log_p.gather(1, at)))
        index.append(torch.where(none, torch.full_like(at, -1), at))
    return torch.cat(values, dim=1), torch.cat(index, dim=1)


def _plain_probs(st):
    case, targets = st["case"], st["targets"]
    z = _plain_scores(st)
    peak = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - peak)
    total = e.sum(dim=1, keepdim=True)
    lse = (peak + torch.log(total)).squeeze(1)
    p = e / total
    log_p = (z - peak) - torch.log(total)                          # z - lse would lose the digits that the peak takes
    entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(dim=1)
    has = targets >= 0
    at = targets.clamp(min=0)[:, None]
    logp = torch.where(has, log_p.gather(1, at).squeeze(1), torch.zeros_like(lse))
    out = {"logp": logp, "entropy": entropy, "lse": lse}
    if case["top"]:
        out["top_logp"], out["top_index"] = _plain_top(z, log_p, case["top"])
    if case["train"]:
        g_logp, g_ent = st["grad_logp"] * has, st["grad_entropy"]
        dz = torch.where(p > 0, p * (-g_logp[:, None] - g_ent[:, None] * (log_p + entropy[:, None])), torch.zeros_like(p))
        dz.scatter_add_(1, at, torch.where(z.gather(1, at) > -float("inf"), g_logp[:, None], torch.zeros_like(peak)))
        dz = dz * case["scale"]
        if case["op"] == "log_probs":
            out["grad_logits"] = dz.to(st["logits"].dtype)
        else:
            out["grad_features"] = (dz @ st["bank"].detach().float()).to(st["features"].dtype)
            out["grad_bank"] = (dz.T @ st["features"].detach().float()).to(st["bank"].dtype)
    return out


def _run_plain(st):
    return _plain_linear(st) if st["case"]["op"] == "linear" else _plain_probs(st)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    train = case["train"]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        size = es * (m * k + n * k + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0))
        if train:
            size += es * (m * n + m * k + n * k + (n if case["bias"] else 0) + (m * n if case["residual"] else 0))
        return {"bytes": size, "flops": (6 if train else 2) * m * n * k}
    rows, cols, k = case["rows"], case["cols"], case["top"]
    size = rows * (8 + 12 + 12 * k) + {"none": 0, "bank": 4 * cols, "rows": 4 * rows * cols}[case["weights"]] + (8 * rows if train else 0)
    if case["op"] == "log_probs":
        size += es * rows * cols * (2 if train else 1)
        return {"bytes": size, "flops": (12 if train else 7) * rows * cols}
    c = case["channels"]
    size += es * c * (rows + cols) * (2 if train else 1)
    return {"bytes": size, "flops": (6 if train else 2) * rows * cols * c}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
_CHUNK = 1 << 27                       # elements of one block of rows in 64 bits (1 GiB)


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_linear(st) if case["op"] == "linear" else _exact_probs(st)


def _exact_linear(st):
    case, d = st["case"], torch.float64
    names = [name for name in ("x", "weight", "bias", "residual") if st[name] is not None]
    m = case["m"]
    step = max(1, _CHUNK // max(case["n"], case["k"]))
    functions = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}
    shared = {name: st[name].detach().to(d).requires_grad_(case["train"]) for name in ("weight", "bias") if name in names}
    parts = {"y": [], "grad_x": [], "grad_residual": []}
    sums = {name: torch.zeros_like(t) for name, t in shared.items()}
    for lo in range(0, m, step):
        own_rows = {name: st[name].detach()[lo:lo + step].to(d).requires_grad_(case["train"]) for name in ("x", "residual") if name in names}
        z = case["alpha"] * (own_rows["x"] @ shared["weight"].t())
        z = z + shared["bias"] if "bias" in shared else z
        y = functions[case["act"]](z)
        y = y + case["beta"] * own_rows["residual"] if "residual" in own_rows else y
        parts["y"].append(y.detach())
        if case["train"]:
            leaves = {**own_rows, **shared}
            grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), st["grad"][lo:lo + step].to(d))))
            for name in own_rows:
                parts["grad_" + name].append(grads[name])
            for name in shared:
                sums[name] += grads[name]
    out = {"y": torch.cat(parts["y"])}
    if case["train"]:
        for name in names:
            out["grad_" + name] = sums[name] if name in sums else torch.cat(parts["grad_" + name])
    return out


def _exact_probs(st):
    case, d, inf = st["case"], torch.float64, float("inf")
    rows, cols, train = case["rows"], case["cols"], case["train"]
    step = max(1, _CHUNK // cols)
    parts, bank_sum = {}, None
    bank = None
    if case["op"] == "bank_log_probs":
        bank = st["bank"].detach().to(d).requires_grad_(train)
        bank_sum = torch.zeros_like(bank)
    for lo in range(0, rows, step):
        block = slice(lo, min(rows, lo + step))
        first = (st["logits"] if bank is None else st["features"]).detach()[block].to(d).requires_grad_(train)
        z = case["scale"] * (first if bank is None else torch.matmul(first, bank.t()))
        gone = None
        if st["weights"] is not None:
            w = st["weights"][block].to(d) if case["weights"] == "rows" else st["weights"].to(d).expand_as(z)
            gone = w == inf
            z = (z - w.masked_fill(gone, 0.0)).masked_fill(gone, -inf)
        lse = torch.logsumexp(z, dim=1)
        log_p = z - lse.unsqueeze(1)
        finite = log_p if gone is None else log_p.masked_fill(gone, 0.0)
        prob = torch.softmax(z, dim=1)
        entropy = -(prob * finite).sum(dim=1)
        targets = st["targets"][block]
        picked = log_p[torch.arange(targets.shape[0], device=z.device), targets.clamp(min=0)]
        logp = torch.where(targets < 0, torch.zeros_like(picked), picked)
        got = {"logp": logp, "entropy": entropy, "lse": lse}
        if case["top"]:
            value, order = torch.sort(z.detach(), dim=1, descending=True, stable=True)
            value, order = value[:, :case["top"]], order[:, :case["top"]]
            got["top_logp"] = value - lse.unsqueeze(1)
            got["top_index"] = order.masked_fill(value == -inf, -1)
        if train:
            leaves = [first] if bank is None else [first, bank]
            grads = torch.autograd.grad((logp, entropy), leaves, (st["grad_logp"][block].to(d), st["grad_entropy"][block].to(d)))
            got["grad_logits" if bank is None else "grad_features"] = grads[0]
            if bank is not None:
                bank_sum += grads[1]
        for key, v in got.items():
            parts.setdefault(key, []).append(v.detach())
    out = {key: torch.cat(v) for key, v in parts.items()}
    if bank is not None and train:
        out["grad_bank"] = bank_sum
    return out
