"""Performance cases of the token-sequence operators: the linear-categorical log-density
(`genjax_amd.linear_categorical`, with its gradient) and the gated delta filter
(`genjax_amd.families.state_space.delta_filter`, its gradient, and its one-token form
`delta_filter_step`).

`run` computes one pass, either in plain torch operations (`own = False`) or through the
framework's entry points (`own = True`); `exact` restates each operator in 64 bits from its
definition, token by token."""
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #
def _score(name, n, vocab, width, dtype):
    return {"name": name, "op": "score", "n": n, "vocab": vocab, "width": width, "dtype": dtype}


def _fit(name, n, vocab, width, dtype):
    return {"name": name, "op": "fit", "n": n, "vocab": vocab, "width": width, "dtype": dtype}


def _seq(name, op, batch, time, kheads, heads, dk, dv, dtype, ragged=False, carried=False):
    return {"name": name, "op": op, "batch": batch, "time": time, "kheads": kheads, "heads": heads, "dk": dk, "dv": dv,
            "dtype": dtype, "ragged": ragged, "carried": carried}


def _step(name, n, kheads, heads, dk, dv, dtype, resampled):
    return {"name": name, "op": "step", "n": n, "kheads": kheads, "heads": heads, "dk": dk, "dv": dv, "dtype": dtype,
            "resampled": resampled}


def listed():
    return [
        # one chain scores its next token: the call's latency and one read of the weights
        _score("score_one_chain", 1, 32000, 1024, "bf16"),
        # the particle count of the small SMC runs, single-precision columns, an odd vocabulary
        _score("score_particles_f32", 200, 50001, 768, "f32"),
        # a whole batch of sequences scored at once
        _score("score_batch", 4096, 128000, 4096, "bf16"),
        # softmax regression inside a gradient move: small and ragged in every size
        _fit("fit_regression_f32", 101, 1003, 65, "f32"),
        # the output layer of a medium sequence model in single precision
        _fit("fit_medium_f32", 1000, 20011, 512, "f32"),
        # the output layer of a large sequence model
        _fit("fit_large", 4096, 128000, 2048, "bf16"),
        # a long sequence read into the memory before sampling starts
        _seq("filter_long", "filter", 1, 8192, 16, 16, 128, 128, "bf16"),
        # a padded batch of unequal sequences that continue from a carried memory, single precision
        _seq("filter_ragged_f32", "filter", 16, 1000, 2, 4, 64, 96, "f32", ragged=True, carried=True),
        # gradient of a short odd sequence (a gradient move over a model's latent embedding)
        _seq("filter_grad_short_f32", "filter_grad", 3, 77, 2, 2, 32, 48, "f32", carried=True),
        # training on a batch of sequences
        _seq("filter_grad_batch", "filter_grad", 4, 2048, 8, 8, 128, 128, "bf16"),
        # one chain takes one token: latency
        _step("step_one_chain", 1, 4, 4, 64, 64, "bf16", False),
        # every particle takes one token right after resampling
        _step("step_particles_resampled", 1000, 4, 8, 128, 128, "bf16", True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["score", "fit", "filter", "filter_grad", "step"])
    dtype = rng.choice(["bf16", "f32"])
    if op in ("score", "fit"):
        # cost of a single-precision product against a bfloat16 one: its operands have three times the bits, so six partial products
        cap = 4096 * 128000 * (4096 if op == "score" else 2048) // (6 if dtype == "f32" else 1)
        while True:
            n, vocab, width = _log_int(rng, 1, 4096), _log_int(rng, 2, 128000), _log_int(rng, 1, 4096)
            if rng.random() < 0.5:
                width = max(64, width // 64 * 64)
            if n * vocab * width <= cap:
                break
        make = _score if op == "score" else _fit
        case = make("", n, vocab, width, dtype)
    elif op == "step":
        kheads = rng.randint(1, 8)
        case = _step("", _log_int(rng, 1, 1000), kheads, kheads * rng.choice([1, 1, 2]), rng.choice([16, 32, 50, 64, 100, 128]),
                     rng.choice([16, 33, 64, 96, 128]), dtype, rng.random() < 0.5)
        while case["n"] * case["heads"] * case["dk"] * case["dv"] > 1000 * 8 * 128 * 128:
            case["n"] = max(1, case["n"] // 2)
    else:
        kheads = rng.randint(1, 8)
        cap = (8192 * 16 if op == "filter" else 4 * 2048 * 8) * 128 * 128
        while True:
            case = _seq("", op, _log_int(rng, 1, 16), _log_int(rng, 1, 8192 if op == "filter" else 2048), kheads,
                        kheads * rng.choice([1, 1, 2]), rng.choice([16, 32, 50, 64, 100, 128]),
                        rng.choice([16, 33, 64, 96, 128]), dtype, rng.random() < 0.5, rng.random() < 0.5)
            if case["batch"] * case["time"] * case["heads"] * case["dk"] * case["dv"] <= cap:
                break
    del case["name"]
    return case


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    def unit(*shape):
        a = normal(*shape)
        return (a / a.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-6)).to(t)

    s = dict(case)
    if case["op"] in ("score", "fit"):
        n, vocab, width = case["n"], case["vocab"], case["width"]
        # features of unit scale against weights that give logits a spread of about two
        s["x"] = normal(n, width, dtype=t)
        s["weight"] = normal(vocab, width, scale=2.0 / width ** 0.5, dtype=t)
        s["bias"] = normal(vocab, scale=0.5, dtype=t)
        s["y"] = torch.randint(0, vocab, (n,), generator=gen, device="cuda", dtype=torch.int32)
        if case["op"] == "fit":
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(True)
            s["upstream"] = normal(n, scale=0.1) + 1.0
        return s

    lead = (case["n"],) if case["op"] == "step" else (case["batch"], case["time"])
    heads, kheads, dk, dv = case["heads"], case["kheads"], case["dk"], case["dv"]
    # unit queries and keys, gains in (0, 1), decays from almost none to fast forgetting
    s["q"], s["k"] = unit(*lead, kheads, dk), unit(*lead, kheads, dk)
    s["v"] = normal(*lead, heads, dv, dtype=t)
    s["log_decay"] = -0.1 * torch.nn.functional.softplus(normal(*lead, heads) * 2.0)
    s["beta"] = torch.sigmoid(normal(*lead, heads))
    if case["op"] == "step":
        n = case["n"]
        s["state"] = normal(n, heads, dk, dv, scale=0.3)
        s["out"] = torch.empty_like(s["state"])
        # systematic resampling leaves sorted ancestors with repeats
        s["ancestors"] = torch.randint(0, n, (n,), generator=gen, device="cuda").sort()[0].to(torch.int32) \
            if case["resampled"] else None
        return s
    batch, time = lead
    s["lengths"] = torch.randint(0, time + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32) \
        if case["ragged"] else None
    s["state"] = normal(batch, heads, dk, dv, scale=0.3) if case["carried"] else None
    if case["op"] == "filter_grad":
        s["leaves"] = [n for n in ("q", "k", "v", "log_decay", "beta", "state") if s[n] is not None]
        for name in s["leaves"]:
            s[name].requires_grad_(True)
        s["d_out"] = normal(batch, time, heads, dv, dtype=t)
        s["d_final"] = normal(batch, heads, dk, dv, scale=0.1)
    return s


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    if s["op"] in ("score", "fit"):
        from genjax_amd import linear_categorical

        lp = linear_categorical.logpdf(s["y"], s["x"], s["weight"], s["bias"])
        if s["op"] == "score":
            return lp
        return (lp.detach(),) + torch.autograd.grad(lp, [s["x"], s["weight"], s["bias"]], s["upstream"])
    from genjax_amd.families.state_space import delta_filter, delta_filter_step

    if s["op"] == "step":
        return delta_filter_step(s["state"], s["q"], s["k"], s["v"], s["log_decay"], s["beta"], ancestors=s["ancestors"],
                                 out=s["out"])
    o, final = delta_filter(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], initial_state=s["state"], lengths=s["lengths"])
    if s["op"] == "filter":
        return o, final
    grads = torch.autograd.grad([o, final], [s[n] for n in s["leaves"]], [s["d_out"], s["d_final"]])
    return (o.detach(), final.detach()) + grads


# ---- plain forms -------------------------------------------------------------
def _run_plain(s):
    if s["op"] in ("score", "fit"):
        return _plain_categorical(s)
    if s["op"] == "step":
        return _plain_step(s)
    names = ("q", "k", "v", "log_decay", "beta", "state")
    leaf = {n: None if s[n] is None else s[n].detach().float() for n in names}
    if s["op"] == "filter":
        o, final = _plain_filter(leaf, s["lengths"])
        return o.to(s["v"].dtype), final
    with torch.enable_grad():
        leaf = {n: None if a is None else a.clone().requires_grad_(True) for n, a in leaf.items()}
        o, final = _plain_filter(leaf, s["lengths"])
        grads = torch.autograd.grad([o, final], [leaf[n] for n in s["leaves"]], [s["d_out"].float(), s["d_final"]])
    return (o.detach().to(s["v"].dtype), final.detach()) + tuple(g.to(s[n].dtype) for g, n in zip(grads, s["leaves"]))


def _plain_categorical(s):
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    y = s["y"].long().unsqueeze(1)
    logits = x @ w.t() + b
    top = logits.max(dim=1, keepdim=True)[0]
    lse = top + (logits - top).exp().sum(dim=1, keepdim=True).log()
    lp = (logits.gather(1, y) - lse).squeeze(1)
    if s["op"] == "score":
        return lp
    g = s["upstream"].unsqueeze(1)
    dl = (logits - lse).exp() * -g
    dl.scatter_add_(1, y, g)
    t = s["x"].dtype
    return lp, (dl @ w).to(t), (dl.t() @ x).to(t), dl.sum(dim=0).to(t)


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular blocks by halves: [[P, 0], [-R c P, R]]."""
    m = a.shape[-1]
    if m == 1:
        return torch.ones_like(a)
    h = m // 2
    p, r = _unit_lower_inverse(a[..., :h, :h]), _unit_lower_inverse(a[..., h:, h:])
    low = -(r @ a[..., h:, :h] @ p)
    return torch.cat([torch.cat([p, torch.zeros_like(low).transpose(-1, -2)], -1), torch.cat([low, r], -1)], -2)


def _plain_filter(a, lengths, chunk=64):
    q, k, v, g, beta, state = (a[n] for n in ("q", "k", "v", "log_decay", "beta", "state"))
    batch, time, heads, dv = v.shape
    dk = k.shape[-1]
    scale = dk ** -0.5
    group = heads // k.shape[2]
    if group > 1:
        q, k = q.repeat_interleave(group, dim=2), k.repeat_interleave(group, dim=2)
    if lengths is not None:
        live = torch.arange(time, device=v.device) < lengths.long().unsqueeze(1)
        wide = live[:, :, None, None]
        q, k, v = (torch.where(wide, t, torch.zeros_like(t)) for t in (q, k, v))
        g, beta = (torch.where(wide[..., 0], t, torch.zeros_like(t)) for t in (g, beta))
    n = (time + chunk - 1) // chunk
    pad = n * chunk - time

    def split(t):
        if pad:
            t = torch.cat([t, torch.zeros_like(t[:, :1]).expand(-1, pad, *t.shape[2:])], 1)
        t = t.reshape(batch, n, chunk, *t.shape[2:]).transpose(2, 3)         # (batch, n, heads, chunk, ...)
        return t.contiguous()

    q, k, v, g, beta = split(q * scale), split(k), split(v), split(g), split(beta)
    total = g.double().cumsum(-1)                                              # 64 bits: differences of long sums
    diff = total.unsqueeze(-1) - total.unsqueeze(-2)
    lower = torch.ones(chunk, chunk, dtype=torch.bool, device=v.device).tril()
    decay = torch.where(lower, diff, torch.full_like(diff, -1e4)).exp().float()
    grow, rest, whole = total.exp().float(), (total[..., -1:] - total).exp().float(), total[..., -1:].exp().float()
    kt = k.transpose(-1, -2).contiguous()
    inner = (k @ kt) * decay * beta.unsqueeze(-1)
    inv = _unit_lower_inverse(torch.where(lower.tril(-1), inner, torch.zeros_like(inner)))
    u = inv @ (v * beta.unsqueeze(-1))
    w = inv @ (k * (beta * grow).unsqueeze(-1))
    reads = (q @ kt) * decay
    late = (k * rest.unsqueeze(-1)).transpose(-1, -2).contiguous()
    q = q * grow.unsqueeze(-1)
    mem = torch.zeros(batch, heads, dk, dv, device=v.device) if state is None else state
    outs = []
    for i in range(n):
        new = u[:, i] - w[:, i] @ mem
        outs.append(q[:, i] @ mem + reads[:, i] @ new)
        mem = mem * whole[:, i].unsqueeze(-1) + late[:, i] @ new
    o = torch.stack(outs, 1).transpose(2, 3).reshape(batch, n * chunk, heads, dv)[:, :time]
    return o.contiguous(), mem


def _plain_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    group = s["heads"] // s["kheads"]
    if group > 1:
        q, k = q.repeat_interleave(group, dim=1), k.repeat_interleave(group, dim=1)
    mem = s["state"] if s["ancestors"] is None else s["state"][s["ancestors"].long()]
    mem = mem * s["log_decay"].exp()[..., None, None]
    u = (v - (mem * k.unsqueeze(-1)).sum(-2)) * s["beta"].unsqueeze(-1)
    mem = mem + k.unsqueeze(-1) * u.unsqueeze(-2)
    o = (mem * q.unsqueeze(-1)).sum(-2) * s["dk"] ** -0.5
    return o.to(s["v"].dtype), mem


# --------------------------------------------------------------------------- #
# what a pass cannot do without
# --------------------------------------------------------------------------- #
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] in ("score", "fit"):
        n, vocab, width = case["n"], case["vocab"], case["width"]
        tensors = e * (n * width + vocab * width + vocab)
        if case["op"] == "score":
            return {"bytes": tensors + 8 * n, "flops": 2 * n * vocab * width}
        return {"bytes": 2 * tensors + 12 * n, "flops": 6 * n * vocab * width}
    heads, kheads, dk, dv = case["heads"], case["kheads"], case["dk"], case["dv"]
    tokens = case["n"] if case["op"] == "step" else case["batch"] * case["time"]
    state = 4 * heads * dk * dv
    once = tokens * (e * (2 * kheads * dk + 2 * heads * dv) + 8 * heads)      # q, k, v, the two gates; o
    per_token = 6 * dk * dv * heads                                             # S^T k, k u^T, S^T q
    if case["op"] == "step":
        return {"bytes": once + 2 * tokens * state, "flops": tokens * per_token}
    carried = state * case["batch"] * (2 if case["carried"] else 1)
    if case["op"] == "filter":
        return {"bytes": once + carried, "flops": tokens * per_token}
    # the gradient reads the upstream of o and of the last state and writes one gradient for each input
    extra = tokens * (e * (2 * kheads * dk + 2 * heads * dv) + 8 * heads)
    return {"bytes": once + extra + 2 * carried, "flops": 3 * tokens * per_token}


# --------------------------------------------------------------------------- #
# the definitions in 64 bits
# --------------------------------------------------------------------------- #
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("score", "fit"):
            return _exact_categorical(s)
        if case["op"] == "step":
            return _exact_step(s)
        return _exact_filter(s)


def _exact_categorical(s):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    n = x.shape[0]
    lp = torch.empty(n, dtype=torch.float64, device="cuda")
    grad = s["op"] == "fit"
    if grad:
        dx, dw, db = torch.empty_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for i in range(0, n, 512):                                   # a few rows at a time
        rows = slice(i, min(n, i + 512))
        logp = torch.log_softmax(torch.addmm(b, x[rows], w.t()), dim=1)
        pick = torch.nn.functional.one_hot(s["y"][rows].long(), w.shape[0]).bool()
        lp[rows] = logp[pick]
        if grad:
            d = (pick.double() - logp.exp()) * s["upstream"][rows].double().unsqueeze(1)
            dx[rows] = torch.mm(d, w)
            dw.addmm_(d.t(), x[rows])
            db += d.sum(0)
    return (lp, dx, dw, db) if grad else lp


def _exact_step(s):
    group = s["heads"] // s["kheads"]
    which = torch.arange(s["heads"], device="cuda") // group
    q, k = s["q"].double()[:, which], s["k"].double()[:, which]
    v, a, beta = s["v"].double(), s["log_decay"].double().exp(), s["beta"].double()
    old = s["state"].double()
    if s["ancestors"] is not None:
        old = old.index_select(0, s["ancestors"].long())
    old = torch.einsum("nh,nhij->nhij", a, old)
    u = beta.unsqueeze(-1) * (v - torch.einsum("nhij,nhi->nhj", old, k))
    new = old + torch.einsum("nhi,nhj->nhij", k, u)
    return torch.einsum("nhij,nhi->nhj", new, q) * s["dk"] ** -0.5, new


def _exact_filter(s):
    """The recurrence one token at a time, and its adjoint one token at a time backwards."""
    batch, time, heads, dk, dv = s["batch"], s["time"], s["heads"], s["dk"], s["dv"]
    grad = s["op"] == "filter_grad"
    if time * (3.0 if grad else 1.0) * 1e-4 > 15 or (grad and 8.0 * batch * time * heads * dk * dv > 6e10):
        return None
    which = torch.arange(heads, device="cuda") // (heads // s["kheads"])
    # (time, batch * heads, ...) so that a token is one contiguous slice
    flat = lambda t: t.double().transpose(0, 1).reshape(time, batch * heads, *t.shape[3:])          # noqa: E731
    q, k, v = flat(s["q"][:, :, which]), flat(s["k"][:, :, which]), flat(s["v"])
    a, beta = flat(s["log_decay"]).exp(), flat(s["beta"])
    on = torch.ones(time, batch, dtype=torch.bool, device="cuda") if s["lengths"] is None else \
        torch.arange(time, device="cuda").unsqueeze(1) < s["lengths"].long()
    on = on.unsqueeze(2).expand(time, batch, heads).reshape(time, batch * heads).double()
    a = a * on + (1.0 - on)
    beta = beta * on
    scale = dk ** -0.5
    mem = torch.zeros(batch * heads, dk, dv, dtype=torch.float64, device="cuda") if s["state"] is None \
        else s["state"].double().reshape(batch * heads, dk, dv)
    kept = torch.empty((time + 1,) + tuple(mem.shape), dtype=torch.float64, device="cuda") if grad else None
    if grad:
        kept[0] = mem
    o = torch.empty(time, batch * heads, dv, dtype=torch.float64, device="cuda")
    for t in range(time):
        mem = mem * a[t, :, None, None]
        u = beta[t, :, None] * (v[t] - torch.bmm(k[t].unsqueeze(1), mem).squeeze(1))
        mem = torch.baddbmm(mem, k[t].unsqueeze(2), u.unsqueeze(1))
        o[t] = torch.bmm(q[t].unsqueeze(1), mem).squeeze(1) * (scale * on[t].unsqueeze(1))
        if grad:
            kept[t + 1] = mem
    back = lambda t: t.reshape(time, batch, heads, *t.shape[2:]).transpose(0, 1)                     # noqa: E731
    final = mem.reshape(batch, heads, dk, dv)
    if not grad:
        return back(o), final
    do = flat(s["d_out"]) * scale * on.unsqueeze(2)
    dmem = s["d_final"].double().reshape(batch * heads, dk, dv).clone()
    dq, dk_, dv_, da, dbeta = (torch.zeros_like(t) for t in (q, k, v, a, beta))
    for t in range(time - 1, -1, -1):
        new, old = kept[t + 1], kept[t] * a[t, :, None, None]
        err = v[t] - torch.bmm(k[t].unsqueeze(1), old).squeeze(1)
        dq[t] = torch.bmm(new, do[t].unsqueeze(2)).squeeze(2)
        dmem = torch.baddbmm(dmem, q[t].unsqueeze(2), do[t].unsqueeze(1))
        du = torch.bmm(k[t].unsqueeze(1), dmem).squeeze(1)
        dk_[t] = torch.bmm(dmem, (beta[t, :, None] * err).unsqueeze(2)).squeeze(2)
        dbeta[t] = (du * err).sum(1)
        dv_[t] = beta[t, :, None] * du
        dk_[t] -= torch.bmm(old, dv_[t].unsqueeze(2)).squeeze(2)
        dmem = torch.baddbmm(dmem, k[t].unsqueeze(2), dv_[t].unsqueeze(1), alpha=-1)
        da[t] = (dmem * old).sum((1, 2))                         # with respect to log a
        dmem = dmem * a[t, :, None, None]
    shared = lambda t: back(t * on.unsqueeze(2)).reshape(batch, time, s["kheads"], -1, dk).sum(3)    # noqa: E731
    grads = {"q": shared(dq), "k": shared(dk_), "v": back(dv_), "log_decay": back(da * on), "beta": back(dbeta * on),
             "state": dmem.reshape(batch, heads, dk, dv)}
    return (back(o), final) + tuple(grads[n] for n in s["leaves"])
