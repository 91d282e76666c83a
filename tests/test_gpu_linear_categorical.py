"""linear_categorical: log-density, gradients and draws against the definition in 64 bits on the same inputs.

Tolerances (per element, from the arithmetic):
 * a logit is a sum of `width` products accumulated in f32; whatever the order, it is off by at most
   2 width 2^-23 sum_k |x_k w_k| (2^-23 a step: the matrix unit may truncate where an addition would round; the factor 2
   covers the f32 operands' partial products left out, 2^-22 of each product) =: E;
 * lse: the exponentials' relative errors (2 E and 2^-22 of expf) and at most 256 additions in a chain, 2^-16 in all;
   the subtraction and the logarithm round once more, 2^-22 of |l| + |lse|;
 * dl = g (onehot - p): p is off by (2 E + 2^-15) p, and dl is rounded to bf16 (2^-8) or split exactly (f32, 2^-22); where
   the forward keeps its exponentials in 11 bits for it (bf16, up to 32 rows or from a width of 512 on) by |g| (2^-11 p + 2^-40) more;
 * dx, dW, db: the products' sums over m terms in f32 add 2 m 2^-23 sum |terms|; the result is rounded once to its type."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def G():
    import genjax_amd

    assert torch.cuda.is_available()
    return genjax_amd


def _inputs(n, vocab, width, dtype, seed=0, bias=True, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(1000 * n + vocab + width + seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")      # noqa: E731
    x, w = r(n, width).to(dtype), (r(vocab, width) * scale / width ** 0.5).to(dtype)
    b = (r(vocab) * 0.5).to(dtype) if bias else None
    y = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    return x, w, b, y, r(n) * 0.1 + 1.0


def _truth(x, w, b, y, up):
    """lp, dx, dW, db in 64 bits and the elementwise bounds of the module's docstring."""
    X, W, u = x.double(), w.double(), up.double().unsqueeze(1)
    vocab, width, n = W.shape[0], W.shape[1], X.shape[0]
    L = X @ W.t() + (0.0 if b is None else b.double())
    lse = torch.logsumexp(L, 1, keepdim=True)
    Y = y.long().clamp(0, vocab - 1).unsqueeze(1)
    lp = (L.gather(1, Y) - lse).squeeze(1)
    mag = X.abs() @ W.abs().t()
    E = 2 * width * 2.0 ** -23 * mag.max(1, keepdim=True)[0]
    lp_tol = (2 * E + 2.0 ** -16 + 2.0 ** -22 * (L.gather(1, Y).abs() + lse.abs())).squeeze(1)
    P = (L - lse).exp()
    D = -P * u
    D.scatter_add_(1, Y, u)
    half = HALF[x.dtype]
    dD = D.abs() * (half if x.dtype == torch.bfloat16 else 2.0 ** -22) + u.abs() * P * (2 * E + 2.0 ** -15)
    if x.dtype == torch.bfloat16 and (n <= 32 or width >= 512):      # formed from what the forward kept
        dD += u.abs() * (P * 2.0 ** -11 + 2.0 ** -40)
    out = {"lp": (lp, lp_tol)}
    dx, dw, db = D @ W, D.t() @ X, D.sum(0)
    out["dx"] = (dx, dD @ W.abs() + 2 * vocab * 2.0 ** -23 * (D.abs() @ W.abs()) + half * dx.abs() + 1e-30)
    out["dw"] = (dw, dD.t() @ X.abs() + 2 * n * 2.0 ** -23 * (D.abs().t() @ X.abs()) + half * dw.abs() + 1e-30)
    out["db"] = (db, dD.sum(0) + 2 * n * 2.0 ** -23 * D.abs().sum(0) + half * db.abs() + 1e-30)
    return out


def _close(name, got, want_tol):
    want, tol = want_tol
    err = (got.double() - want).abs()
    worst = (err / tol).max().item()
    assert got.shape == want.shape and worst <= 1.0, f"{name}: {worst:.3g} times its bound (error {err.max().item():.3g})"


def _grads(G, x, w, b, y, up):
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b) if t is not None]
    lp = G.linear_categorical.logpdf(y, *leaves)
    return (lp.detach(),) + torch.autograd.grad(lp, leaves, up)


SIZES = [(1, 1, 1), (1, 2, 7), (3, 5, 64), (5, 257, 65), (64, 256, 64), (65, 300, 128), (130, 70, 1000), (17, 4099, 520),
         (257, 511, 192), (33, 2560, 8), (300, 33000, 64), (1000, 20011, 72), (4, 1500, 4096)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,vocab,width", SIZES)
def test_logpdf_and_gradients(G, n, vocab, width, dtype):
    x, w, b, y, up = _inputs(n, vocab, width, TYPES[dtype])
    t = _truth(x, w, b, y, up)
    _close("lp without a gradient", G.linear_categorical.logpdf(y, x, w, b), t["lp"])
    for name, got in zip(("lp", "dx", "dw", "db"), _grads(G, x, w, b, y, up)):
        _close(name, got, t[name])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_bias_strided_rows_and_partial_gradients(G, dtype):
    t = TYPES[dtype]
    n, vocab, width = 70, 900, 128
    wide_x, wide_w, _, y, up = _inputs(n, vocab, 2 * width + 5, t, bias=False)
    x, w = wide_x[:, 3:3 + width], wide_w[:, 1:1 + width]                  # spaced, misaligned rows
    want = _truth(x, w, None, y, up)
    _close("lp", G.linear_categorical.logpdf(y, x, w), want["lp"])
    for name, leaf in (("dx", 0), ("dw", 1)):                              # one gradient at a time
        args = [x.detach(), w.detach()]
        args[leaf] = args[leaf].clone().requires_grad_(True)
        lp = G.linear_categorical.logpdf(y, *args)
        _close(name, torch.autograd.grad(lp, args[leaf], up)[0], want[name])
    xt = wide_x[:, :width].t().contiguous().t()                            # columns contiguous: copied inside
    _close("lp of a transposed x", G.linear_categorical.logpdf(y, xt, w), _truth(xt, w, None, y, up)["lp"])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [3, 200])
def test_masked_entries_and_empty_rows(G, n, dtype):
    x, w, b, y, up = _inputs(n, 700, 64, TYPES[dtype])
    b[::3] = -float("inf")
    y = y // 3 * 3 + 1                                     # an entry that is left
    y[y >= 700] = 1
    t = _truth(x, w, b, y, up)
    for name, got in zip(("lp", "dx", "dw", "db"), _grads(G, x, w, b, y, up)):
        _close(name, got, t[name])
        assert torch.isfinite(got).all()
    y0 = torch.zeros_like(y)                               # a masked entry has density zero
    assert torch.equal(G.linear_categorical.logpdf(y0, x, w, b), torch.full((n,), -float("inf"), device="cuda"))
    low = torch.full_like(b, torch.finfo(b.dtype).min)     # masks of the type's lowest value: finite and normalised
    low[5] = 0.0
    lp = G.linear_categorical.logpdf(torch.full_like(y, 5), x, w, low)
    assert torch.equal(lp, torch.zeros_like(lp))
    none = torch.full_like(b, -float("inf"))               # no entry left
    assert torch.isnan(G.linear_categorical.logpdf(y, x, w, none)).all()


def test_values_outside_the_vocabulary_take_the_nearest_entry(G):
    from genjax_amd import backend as B

    x, w, b, _, _ = _inputs(6, 40, 64, torch.float32)
    y = torch.tensor([-5, 0, 39, 40, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    got = G.linear_categorical.logpdf(y, x, w, b)
    assert torch.equal(got, G.linear_categorical.logpdf(y.clamp(0, 39), x, w, b))
    ref = B.categorical_logpdf(y, x @ w.t() + b)           # the same rule as categorical's
    np.testing.assert_allclose(got.cpu().numpy(), ref.cpu().numpy(), atol=1e-4)


def test_shared_rows_scalars_and_empty_batches(G):
    x, w, b, y, up = _inputs(5, 90, 64, torch.float32)
    one = G.linear_categorical.logpdf(y[0], x[0], w, b)
    assert one.dim() == 0
    _close("one", one.reshape(1), tuple(v[:1] for v in _truth(x, w, b, y, up)["lp"]))
    same = x[:1].expand(5, 64)
    _close("shared x", G.linear_categorical.logpdf(y, x[0], w, b), _truth(same, w, b, y, up)["lp"])
    _close("shared y", G.linear_categorical.logpdf(y[0], x, w, b), _truth(x, w, b, y[:1].expand(5), up)["lp"])
    leaf = x[0].clone().requires_grad_(True)               # a shared row collects the gradient of every value
    lp = G.linear_categorical.logpdf(y, leaf, w, b)
    want, tol = _truth(same, w, b, y, up)["dx"]
    _close("dx of a shared row", torch.autograd.grad(lp, leaf, up)[0], (want.sum(0), tol.sum(0) + 2.0 ** -20 * want.abs().sum(0)))
    e = torch.empty(0, 64, device="cuda", requires_grad=True)
    w2 = w.clone().requires_grad_(True)
    lp = G.linear_categorical.logpdf(y[:0], e, w2, b)
    assert lp.shape == (0,)
    gx, gw = torch.autograd.grad(lp.sum(), (e, w2))
    assert gx.shape == (0, 64) and torch.equal(gw, torch.zeros_like(w))


def test_gradient_against_differences(G):
    x, w, b, y, up = _inputs(40, 333, 24, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(3)
    for i, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, generator=g, device="cuda")
        d = d / d.norm()
        h = 2.0 ** -6
        args = [x, w, b]
        f = []
        for s in (h, -h):
            args[i] = t + s * d
            f.append((G.linear_categorical.logpdf(y, *args) * up).sum().double())
        num = ((f[0] - f[1]) / (2 * h)).item()
        ana = (_grads(G, x, w, b, y, up)[1 + i].double() * d.double()).sum().item()
        # forty log-densities of ~2^3, each off by up to 2^-16: 2^-7 of difference quotient at worst; h^2 terms below that
        assert abs(num - ana) <= 2.0 ** -6 * max(1.0, abs(ana)), (i, num, ana)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,vocab,width", [(1, 3, 64), (50, 777, 40), (300, 33000, 64)])
def test_draws(G, n, vocab, width, dtype):
    """The draw maximises l + Gumbel over categorical's noise: where the 64-bit runner-up is further away than the
    logits' error, the entry is that one; with the framework's own logits it is categorical's draw."""
    from genjax_amd import backend as B

    x, w, b, y, up = _inputs(n, vocab, width, TYPES[dtype])
    key = G.key(7)
    got = B.sample_linear_categorical(key, x, w, b)
    u = B.random_uniform(key, n * vocab, 1.17549435e-38, 1.0).double().reshape(n, vocab)
    z = x.double() @ w.double().t() + b.double() - (-u.log()).log()
    top = z.topk(2, dim=1)
    clear = (top[0][:, 0] - top[0][:, 1]) > 1e-3
    assert clear.float().mean() > 0.9 and torch.equal(got.long()[clear], top[1][:, 0][clear])
    assert ((z.gather(1, got.long().unsqueeze(1)).squeeze(1) - top[0][:, 0]).abs() <= 1e-3).all()
    cat = B.sample_categorical(key, (x.double() @ w.double().t() + b.double()).float())
    assert torch.equal(cat[clear], got[clear])
    b2 = torch.full_like(b, -float("inf"))                 # masked entries are never drawn
    b2[vocab // 2] = 0.0
    assert (B.sample_linear_categorical(key, x, w, b2) == vocab // 2).all()


def test_draw_frequencies_and_gfi(G):
    from genjax_amd import gen, linear_categorical, seed
    from genjax_amd.core import batched

    x, w, b, _, _ = _inputs(1, 6, 8, torch.float32)

    @gen
    def model(x, w, b):
        return linear_categorical(x, w, b) @ "token"

    n = 20000
    with batched(n):
        tr = seed(model.simulate)(G.key(1), x[0], w, b)
    tok = tr.get_choices()["token"]
    assert tok.shape == (n,) and tok.dtype == torch.int32
    p = torch.softmax((x @ w.t() + b)[0], 0)
    freq = torch.bincount(tok.long(), minlength=6) / n
    assert ((freq - p).abs() <= 6 * (p * (1 - p) / n).sqrt() + 1e-6).all()      # six standard errors
    lp, _ = model.assess({"token": tok}, x[0], w, b)
    np.testing.assert_allclose(tr.get_score().cpu().numpy(), -lp.cpu().numpy(), rtol=0, atol=0)


def test_hmc_over_latent_features(G):
    """The gradient move differentiates through the density: hmc on a latent feature row per chain runs and its
    log-density gradient is the 64-bit one."""
    from genjax_amd import gen, linear_categorical, normal, seed, sel
    from genjax_amd.core import batched
    from genjax_amd.inference import hmc
    from genjax_amd.inference.mcmc import _SelectedDensity

    _, w, b, y, _ = _inputs(1, 50, 2, torch.float32)

    @gen
    def model(w, b):
        h0 = normal(0.0, 1.0) @ "h0"
        h1 = normal(0.0, 1.0) @ "h1"
        linear_categorical(torch.stack([h0, h1], -1), w, b) @ "token"

    n = 64
    with batched(n):
        tr, _ = seed(model.generate)(G.key(3), {"token": y[0]}, w, b)
        d = _SelectedDensity(tr, sel("h0") | sel("h1"))
        _, grads = d.logp(d.q0, True)
        x = torch.stack(d.q0, -1)
        up = torch.ones(n, device="cuda")
        want, tol = _truth(x, w, b, y[:1].expand(n), up)["dx"]
        _close("gradient", torch.stack(grads, -1), (want - x.double(), tol + 2.0 ** -20 * (want.abs() + x.abs())))
        out = seed(lambda t: hmc(t, sel("h0") | sel("h1"), 0.1, 5))(G.key(4), tr)
    assert torch.isfinite(out.get_choices()["h0"]).all()


def test_weights_beyond_32_bit_offsets(G):
    """vocab x width passes 2^31 elements; the last entries' logits and gradients come from the right rows."""
    n, vocab, width = 2, (1 << 20) + 300, 2048
    w = torch.zeros(vocab, width, dtype=torch.bfloat16, device="cuda")
    w[-300:] = torch.randn(300, width, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16) * 0.1
    x = torch.randn(n, width, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(torch.bfloat16)
    y = torch.tensor([vocab - 1, vocab - 150], dtype=torch.int32, device="cuda")
    tail = x.double() @ w[-300:].double().t()
    lse = torch.logsumexp(torch.cat([tail, torch.full((n, 1), float(np.log(vocab - 300)), device="cuda", dtype=torch.float64)], 1), 1)
    want = tail[torch.arange(n), (y - (vocab - 300)).long()] - lse
    leaf = w.requires_grad_(True)
    lp = G.linear_categorical.logpdf(y, x, leaf)
    assert ((lp.double() - want).abs() <= 2.0 ** -10).all()
    dw = torch.autograd.grad(lp.sum(), leaf)[0]
    d = -(tail - lse.unsqueeze(1)).exp()
    d[torch.arange(n), (y - (vocab - 300)).long()] += 1.0
    err = (dw[-300:].double() - d.t() @ x.double()).abs()
    assert (err <= 2.0 ** -6 * (d.abs().t() @ x.double().abs()) + 1e-9).all()
    p = (-lse).exp().unsqueeze(1)                          # every entry with zero weights has this probability
    zero = (p * x.double()).sum(0)
    assert ((dw[:1000].double() + zero).abs() <= 2.0 ** -6 * (p * x.double().abs()).sum(0)).all()


def test_streams_and_captured_graphs(G):
    """A call on a side stream; two graphs captured from calls of different sizes, replayed in turn with new inputs,
    each against the eager result (forward, gradient and draw)."""
    from genjax_amd import backend as B

    side = torch.cuda.Stream()
    sets = []
    for n, vocab, width in ((70, 1000, 96), (33, 2500, 64)):
        x, w, b, y, up = _inputs(n, vocab, width, torch.bfloat16)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            lp, lse = B.linear_categorical_logpdf(y, x, w, b)
        side.synchronize()
        assert torch.equal(lp, B.linear_categorical_logpdf(y, x, w, b)[0])

        def call(x=x, w=w, b=b, y=y, up=up):
            lp, lse = B.linear_categorical_logpdf(y, x, w, b)
            return [lp] + B.linear_categorical_grad(y, x, w, b, lse, up) + [B.sample_linear_categorical(G.key(1), x, w, b)]

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call()
        sets.append((graph, outs, call, x, up))
    for turn in range(4):
        for graph, outs, call, x, up in sets:
            x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(turn)).to(x.dtype))
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(outs, want))


def test_same_bits_on_every_call(G):
    x, w, b, y, up = _inputs(300, 20011, 256, torch.bfloat16)
    first = _grads(G, x, w, b, y, up)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, _grads(G, x, w, b, y, up)))


# ---- what the forward keeps for the gradient ---------------------------------
# Up to 32 rows, and from a width of 128 (f32) or 512 (bf16) on, the gradient is formed from the forward's exponentials.  In
# f32 they are kept as they are: exp(l - base) and exp(base - lse) share the error that exp(l - lse) had.  In bf16 they are
# kept in 11 bits (2^-11, and 2^-40 of the block's largest absolutely), before dl is rounded as everywhere.
def _check_kept(G, n, vocab, width, dtype, bias=True):
    from genjax_amd import backend as B

    x, w, b, y, up = _inputs(n, vocab, width, dtype, bias=bias)
    t = _truth(x, w, b, y, up)
    args = [a for a in (x, w, b) if a is not None]
    lp, lse, kept = B.linear_categorical_logpdf(y, *args, keep=True)
    assert kept is not None
    plain, lse2 = B.linear_categorical_logpdf(y, *args)
    _close("lp", lp, t["lp"])
    _close("lp of the call that keeps nothing", plain, t["lp"])      # (its tiles may be others)
    assert torch.equal(lp.isnan(), plain.isnan()) and lse.shape == lse2.shape
    got = B.linear_categorical_grad(y, x, w, b, lse, up, kept=kept)
    again = B.linear_categorical_grad(y, x, w, b, lse, up, kept=kept)          # what is kept is only read
    for name, g, g2 in zip(("dx", "dw", "db"), got, again):
        if g is not None:
            _close(name, g, t[name])
            assert torch.equal(g, g2)
    for want in ((True, False, False), (False, True, False), (False, False, b is not None)):
        part = B.linear_categorical_grad(y, x, w, b, lse, up, want=want, kept=kept)
        for wanted, p, g in zip(want, part, got):
            assert torch.equal(p, g) if wanted else p is None


@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 70, 33), (16, 1000, 100), (17, 9000, 65), (32, 129, 1100), (33, 2, 128), (33, 300, 257), (64, 257, 300), (130, 4099, 512), (200, 50001, 256), (1000, 140001, 256)])
def test_gradient_from_what_the_forward_kept_f32(G, n, vocab, width):
    _check_kept(G, n, vocab, width, torch.float32, bias=vocab != 300)


@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 70, 33), (16, 1000, 100), (17, 9000, 65), (32, 129, 2100), (33, 2, 512), (33, 300, 1030), (100, 511, 576), (257, 70000, 1024), (4000, 70001, 1024)])
def test_gradient_from_what_the_forward_kept_bf16(G, n, vocab, width):
    _check_kept(G, n, vocab, width, torch.bfloat16, bias=vocab != 300)


def test_kept_rows_without_an_entry_and_masked_entries(G):
    """Entries with a bias of -inf keep a gradient of 0, values there a log-density of -inf, rows without any entry are NaN;
    a graph that is replayed and an eager backward in between agree."""
    n, vocab, width = 70, 600, 256
    x, w, b, y, up = _inputs(n, vocab, width, torch.float32)
    b[100:500] = -float("inf")
    y = torch.where((y >= 100) & (y < 500), 5, y).to(torch.int32)
    t = _truth(x, w, b, y, up)
    for name, got in zip(("lp", "dx", "dw", "db"), _grads(G, x, w, b, y, up)):
        _close(name, got, t[name])
        if name in ("dw", "db"):
            assert not got[100:500].any()
    y2 = y.clone()
    y2[3] = 200
    lp, dx, dw, db = _grads(G, x, w, b, y2, up)
    assert lp[3] == -float("inf") and torch.isfinite(dx).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()
    lp, *_ = _grads(G, x, w, torch.full_like(b, -float("inf")), y, up)
    assert torch.isnan(lp).all()


def test_two_backwards_and_a_large_shift(G):
    """retain_graph: the second backward gives the same; logits near 300 (a bias common to all) change nothing."""
    x, w, b, y, up = _inputs(90, 700, 320, torch.float32)
    leaves = [a.clone().requires_grad_(True) for a in (x, w, b + 300.0)]
    lp = G.linear_categorical.logpdf(y, *leaves)
    one = torch.autograd.grad(lp, leaves, up, retain_graph=True)
    two = torch.autograd.grad(lp, leaves, up)
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    t = _truth(x, w, b + 300.0, y, up)
    # a logit near 300 is rounded to 2^-24 of it after the bias is added: E grows by 2^-24 * 300 < 2^-15, in p as in dl
    P = torch.softmax(x.double() @ w.double().t() + b.double(), 1) * up.double().abs().unsqueeze(1) * 2.0 ** -14
    for name, got, more in zip(("dx", "dw", "db"), one, (P @ w.double().abs(), P.t() @ x.double().abs(), P.sum(0))):
        _close(name, got, (t[name][0], t[name][1] + more))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,vocab,width", [(1500, 7, 96), (700, 300, 500), (4000, 1, 33), (1000, 2000, 64)])
def test_many_rows_of_few_values(G, n, vocab, width, dtype):
    """The rows of dW's sums shared out over workgroups, many of them with the same value."""
    x, w, b, y, up = _inputs(n, vocab, width, TYPES[dtype])
    t = _truth(x, w, b, y, up)
    one = _grads(G, x, w, b, y, up)
    for name, got, again in zip(("lp", "dx", "dw", "db"), one, _grads(G, x, w, b, y, up)):
        _close(name, got, t[name])
        assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", [torch.int64, torch.float32, torch.uint8])
def test_values_of_other_types(G, dtype):
    x, w, b, y, _ = _inputs(6, 9, 16, torch.float32)
    far = torch.tensor([-5, 0, 8, 9, 2 ** 32 + 3, -2 ** 40] if dtype == torch.int64 else [0, 1, 2, 8, 9, 200], device="cuda").to(dtype)
    near = far.long().clamp(0, 8).to(torch.int32)
    assert torch.equal(G.linear_categorical.logpdf(far, x, w, b), G.linear_categorical.logpdf(near, x, w, b))


@pytest.mark.parametrize("n", [129, 150, 200, 208, 209])
def test_rows_of_one_wide_tile(G, n):
    """f32 density and draw around the row counts that one tile holds, at a vocabulary where it is taken."""
    from genjax_amd import backend as B

    x, w, b, y, up = _inputs(n, 52003, 100, torch.float32)
    t = _truth(x, w, b, y, up)
    _close("lp", G.linear_categorical.logpdf(y, x, w, b), t["lp"])
    flat = torch.zeros_like(w)
    flat[:, 0] = torch.linspace(-1, 1, 52003, device="cuda")
    peak = torch.where(torch.arange(52003, device="cuda") == 11000, 200.0, 0.0)
    assert (B.sample_linear_categorical(G.key(2), x, flat, peak) == 11000).all()
    key = G.key(7)
    ours = B.sample_linear_categorical(key, x, w, b)
    # the same draws as categorical's over the rounded logits, but where two entries lie within the logits' error
    ref = B.sample_categorical(key, (x.double() @ w.double().t() + b.double()).float())
    assert (ours == ref).float().mean() >= 0.98


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,vocab,width", [(2, 326, 3867), (1, 1, 4096), (32, 3000, 4100), (500, 31, 3000), (64, 1500, 1024), (40, 5000, 800),
                                           (129, 700, 2048), (2000, 3, 1000)])
def test_few_tiles_and_long_rows(G, n, vocab, width, dtype):
    """The products whose reduction is cut along the width: log-density, gradients (kept or formed again), draws."""
    from genjax_amd import backend as B

    x, w, b, y, up = _inputs(n, vocab, width, TYPES[dtype])
    if vocab > 2:
        b[1] = -float("inf")
        y[y == 1] = 0
    t = _truth(x, w, b, y, up)
    one = _grads(G, x, w, b, y, up)
    for name, got, again in zip(("lp", "dx", "dw", "db"), one, _grads(G, x, w, b, y, up)):
        _close(name, got, t[name])
        assert torch.equal(got, again)
    _close("lp without a gradient", G.linear_categorical.logpdf(y, x, w, b), t["lp"])
    lp, lse = B.linear_categorical_logpdf(y, x, w, b)
    for name, got in zip(("dx", "dw", "db"), B.linear_categorical_grad(y, x, w, b, lse, up)):      # nothing kept
        _close(name + " formed again", got, t[name])
    key = G.key(11)
    got = B.sample_linear_categorical(key, x, w, b)
    u = B.random_uniform(key, n * vocab, 1.17549435e-38, 1.0).double().reshape(n, vocab)
    z = x.double() @ w.double().t() + b.double() - (-u.log()).log()
    best = z.max(dim=1)[0]
    # the logits are off by E = 2 width 2^-23 sum |x w| at most, the noise by some units of 2^-24 of at most ~20
    E = 2 * width * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).max(1)[0]
    assert (best - z.gather(1, got.long().unsqueeze(1)).squeeze(1) <= 2 * E + 1e-4).all()
    assert vocab < 2 or (got != 1).all() or vocab <= 2


def _far_below(G, n, vocab, width, dtype, shift, masked=None):
    """Gradients where every logit lies `shift` below 0, entries `masked` taken out: a common shift changes no probability."""
    x, w, b, y, up = _inputs(n, vocab, width, dtype)
    b = (b.float() + shift).to(dtype)
    if masked is not None:
        b[masked] = -float("inf")
        y = torch.full_like(y, vocab - 1)
    t = _truth(x, w, b, y, up)
    # a logit of this size is rounded to 2^-24 of it after the bias is added: dl moves by twice that of p
    P = torch.softmax(x.double() @ w.double().t() + b.double(), 1) * up.double().abs().unsqueeze(1) * 2.0 ** -23 * (abs(shift) + 16)
    more = (0.0, P @ w.double().abs(), P.t() @ x.double().abs(), P.sum(0))
    for name, got, m in zip(("lp", "dx", "dw", "db"), _grads(G, x, w, b, y, up), more):
        assert torch.isfinite(got).all(), name
        _close(name, got, (t[name][0], t[name][1] + m))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 17, 32, 70])
@pytest.mark.parametrize("vocab", [1, 7, 16, 33, 65, 257, 1040])
def test_gradient_of_logits_far_below_zero(G, n, vocab, dtype):
    """Entries behind the vocabulary stand in the products' tiles beside logits near -300."""
    _far_below(G, n, vocab, 64 if n <= 32 else 576, TYPES[dtype], -300.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,width", [(1, 64), (32, 64), (70, 576), (300, 576), (300, 64)])
def test_gradient_beside_masked_blocks_far_below_zero(G, n, width, dtype):
    """Whole blocks of entries without one that is left, logits near -120 elsewhere."""
    _far_below(G, n, 1300, width, TYPES[dtype], -120.0, slice(100, 1000))


@pytest.mark.parametrize("n,vocab,width,dtype", [(4000, 70001, 64, "bf16"), (2000, 70001, 65, "f32"), (1000, 560001, 130, "f32")])
def test_gradient_formed_again_in_pieces_of_the_vocabulary(G, n, vocab, width, dtype):
    """Nothing is kept (too narrow, or above 2 GiB) and dl passes 512 MiB: each piece adds to dx, fills its own rows of dW and
    db, and holds the values of its own entries."""
    from genjax_amd import backend as B

    t = TYPES[dtype]
    x, w, b, y, up = _inputs(n, vocab, width, t)
    assert B.linear_categorical_logpdf(y, x, w, b, keep=True)[2] is None
    half = -(-(-(-vocab // 2)) // 256) * 256                # where the second of two equal pieces begins
    for i, v in enumerate((0, half - 1, half, half + 1, vocab - 1)):
        y[7 * i:7 * i + 7] = v
    want = _truth(x, w, b, y, up)
    for name, got in zip(("lp", "dx", "dw", "db"), _grads(G, x, w, b, y, up)):
        _close(name, got, want[name])


@pytest.mark.parametrize("n", [40, 70])
def test_packed_weights_in_pieces(G, n):
    """bf16 weights whose rows are packed for the tile loader, 547 MiB of them: two pieces."""
    from genjax_amd import backend as B

    vocab, width = 140001, 2000
    x, w, b, y, up = _inputs(n, vocab, width, torch.bfloat16)
    half = -(-(-(-vocab // 2)) // 256) * 256
    y[:3] = torch.tensor([half - 1, half, vocab - 1], dtype=torch.int32, device="cuda")
    want = _truth(x, w, b, y, up)
    for name, got in zip(("lp", "dx", "dw", "db"), _grads(G, x, w, b, y, up)):
        _close(name, got, want[name])
    lp, lse = B.linear_categorical_logpdf(y, x, w, b)
    _close("lp that keeps nothing", lp, want["lp"])
    for name, got in zip(("dx", "dw", "db"), B.linear_categorical_grad(y, x, w, b, lse, up)):
        _close(name + " formed again", got, want[name])
    key = G.key(5)
    got = B.sample_linear_categorical(key, x, w, b)
    u = B.random_uniform(key, n * vocab, 1.17549435e-38, 1.0).double().reshape(n, vocab)
    z = x.double() @ w.double().t() + b.double() - (-u.log()).log()
    E = 2 * width * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).max(1)[0]
    assert (z.max(dim=1)[0] - z.gather(1, got.long().unsqueeze(1)).squeeze(1) <= 2 * E + 1e-4).all()
    assert (got >= half).any() and (got < half).any()


@pytest.mark.parametrize("dtype,vocab", [("bf16", 1 << 19), ("f32", 1 << 18)])
def test_more_tiles_than_a_row_of_the_grid(G, dtype, vocab):
    """2^20 rows: the product's tiles along one axis would pass 2^32 threads."""
    n, width = 1 << 20, 32
    x, w, b, y, _ = _inputs(n, vocab, width, TYPES[dtype])
    lp = G.linear_categorical.logpdf(y, x, w, b)
    for i in (0, 1000, n // 2 - 1, n // 2, n - 3):
        part = slice(i, i + 3)
        _close("lp", lp[part], _truth(x[part], w, b, y[part], torch.ones(3, device="cuda"))["lp"])
    assert torch.isfinite(lp).all() and (lp < 0).all()


def test_draws_of_a_shape(G):
    """sample_shape as categorical takes it: that many draws from one row; anything else is refused, not ignored."""
    from genjax_amd import backend as B

    x, w, b, _, _ = _inputs(3, 6, 8, torch.float32)
    draw = lambda *a, **k: G.seed(lambda: G.linear_categorical.sample(*a, **k))(G.key(1))      # noqa: E731
    assert draw(x[0], w, b, sample_shape=(50,)).shape == (50,) and draw(x[0], w, b).shape == () and draw(x, w, b).shape == (3,)
    logits = x[0] @ w.t() + b
    ref = G.seed(lambda: G.categorical.sample(logits, sample_shape=(50,)))(G.key(1))
    assert ref.shape == (50,) and len(set(draw(x[0], w, b, sample_shape=(50,)).tolist())) > 1
    for bad in (dict(x=x, sample_shape=(50,)), dict(x=x[0], sample_shape=(5, 10))):
        with pytest.raises(B.GjxError, match="sample_shape"):
            draw(bad["x"], w, b, sample_shape=bad["sample_shape"])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,vocab,width", [(20, 3000, 64), (100, 9000, 640)])
def test_a_gradient_without_kept_exponentials(G, n, vocab, width, dtype):
    """keep=False: the same bounds, and between forward and backward no more than the outputs and the inputs are held."""
    x, w, b, y, up = _inputs(n, vocab, width, TYPES[dtype])
    want = _truth(x, w, b, y, up)
    held = []
    for keep in (True, False):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        lp = G.linear_categorical.logpdf(y, *leaves, keep=keep)
        held.append(torch.cuda.memory_allocated() - before)
        _close("lp", lp.detach(), want["lp"])
        for name, got in zip(("dx", "dw", "db"), torch.autograd.grad(lp, leaves, up)):
            _close(name, got, want[name])
    assert held[0] >= n * vocab * (2 if dtype == "bf16" else 4) and held[1] <= 4096
    tr, _ = G.seed(lambda: G.linear_categorical.generate(y, x, w, b, keep=False))(G.key(0))      # through the interface, too
    assert torch.equal(tr.get_score(), -G.linear_categorical.logpdf(y, x, w, b))


def test_no_value_of_a_shared_row(G):
    x, w, b, y, _ = _inputs(1, 6, 8, torch.float32)
    for row in (x[0], x):
        leaves = [t.clone().requires_grad_(True) for t in (row, w, b)]
        assert G.linear_categorical.logpdf(y[:0], row, w, b).shape == (0,)
        lp = G.linear_categorical.logpdf(y[:0], *leaves)
        assert lp.shape == (0,)
        for g, t in zip(torch.autograd.grad(lp.sum(), leaves), leaves):
            assert torch.equal(g, torch.zeros_like(t))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,vocab,width", [(100000, 50, 64), (300, 100, 2048)])
def test_captured_gradient_of_a_shared_row(G, n, vocab, width, dtype):
    """The row's gradient is a sum over all values; every replay against the eager result."""
    x, w, _, y, up = _inputs(n, vocab, width, TYPES[dtype])
    leaf = x[0].clone().requires_grad_(True)

    def grad():
        return torch.autograd.grad(G.linear_categorical.logpdf(y, leaf, w), leaf, up)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grad()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = grad()
    for turn in range(5):
        with torch.no_grad():
            leaf.copy_(torch.randn(width, device="cuda", generator=torch.Generator("cuda").manual_seed(turn)))
        graph.replay()
        want = grad()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
