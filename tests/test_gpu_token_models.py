"""delta_filter, delta_filter_step and linear_categorical together, as a token model uses them: a state-space model whose
state is a matrix of regression weights and whose observations are tokens of a vocabulary.

Tolerances: the truth takes the same inputs in 64 bits, and each operator's own bounds (its own tests) are carried through
the next.  An o entry is off by at most e = 2^-15 max |o| (f32); a logit is a sum of `width` products of o with a weight
row, so it moves by at most e sum_k |w_k|, and the log-density by twice the largest such move, besides the density's own
2 E + 2^-16 + 2^-22 (|logit| + |lse|) with E = 2 width 2^-23 max sum |x w|.  Sums over T tokens add T of these."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def G():
    import genjax_amd

    assert torch.cuda.is_available()
    return genjax_amd


class _Model:
    """Token embeddings -> (q, k, v, gates), the filter, and a linear read-out over the vocabulary; all weights f32."""

    def __init__(self, vocab=37, kheads=1, heads=2, dk=24, dv=16, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=gen, device="cuda")        # noqa: E731
        unit = lambda t: t / t.norm(dim=-1, keepdim=True)                  # noqa: E731
        self.vocab, self.kheads, self.heads, self.dk, self.dv = vocab, kheads, heads, dk, dv
        self.q, self.k, self.v = unit(r(vocab, kheads, dk)), unit(r(vocab, kheads, dk)), r(vocab, heads, dv)
        self.g, self.beta = -0.1 * torch.rand(vocab, heads, generator=gen, device="cuda"), torch.sigmoid(r(vocab, heads))
        self.w, self.b = r(vocab, heads * dv) * 0.4, r(vocab) * 0.2

    def tables(self):
        return self.q, self.k, self.v, self.g, self.beta

    def inputs(self, tokens):
        return [t[tokens.long()] for t in self.tables()]

    def state(self, n):
        return torch.zeros(n, self.heads, self.dk, self.dv, device="cuda")


def _truth(m, y, tables, w, b):
    """Per-token log-densities of whole sequences y (batch, T + 1) in 64 bits, differentiable -> ((batch, T), bounds)."""
    q, k, v, g, beta = (t[y[:, :-1].long()] for t in tables)
    group = m.heads // m.kheads
    q, k = q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)
    mem = torch.zeros(y.shape[0], m.heads, m.dk, m.dv, dtype=torch.float64, device="cuda")
    outs = []
    for t in range(y.shape[1] - 1):
        mem = mem * g[:, t].exp()[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (mem * k[:, t, :, :, None]).sum(2))
        mem = mem + k[:, t, :, :, None] * u[:, :, None, :]
        outs.append(m.dk ** -0.5 * (mem * q[:, t, :, :, None]).sum(2))
    o = torch.stack(outs, 1).flatten(2)
    logits = o @ w.t() + b
    at = y[:, 1:].long().unsqueeze(-1)
    lse = torch.logsumexp(logits, -1, keepdim=True)
    with torch.no_grad():
        e = 2.0 ** -15 * o.abs().max() * w.abs().sum(-1).max()
        big = 2 * o.shape[-1] * 2.0 ** -23 * (o.abs() @ w.abs().t()).max()
        tol = 2 * e + 2 * big + 2.0 ** -16 + 2.0 ** -22 * (logits.abs().max() + lse.abs().max())
    return (logits.gather(-1, at) - lse).squeeze(-1), tol.item()


def _whole(G, m, y, tables, w, b):
    """The same through the library: one filter over the sequences, one density over all their tokens."""
    from genjax_amd.families.state_space import delta_filter

    o, _ = delta_filter(*(t[y[:, :-1].long()] for t in tables))
    rows = o.flatten(2).flatten(0, 1)
    return G.linear_categorical.logpdf(y[:, 1:].reshape(-1), rows, w, b).view(y.shape[0], -1)


def _sequences(m, batch, time, seed=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, m.vocab, (batch, time + 1), generator=gen, device="cuda", dtype=torch.int32)


def test_whole_sequences_and_training_gradient(G):
    m = _Model()
    y = _sequences(m, 3, 97)
    leaves = [t.clone().requires_grad_(True) for t in (*m.tables(), m.w, m.b)]
    lp = _whole(G, m, y, leaves[:5], *leaves[5:])
    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    want, tol = _truth(m, y, exact[:5], *exact[5:])
    assert ((lp - want).abs() <= tol).all()
    got = torch.autograd.grad(lp.sum(), leaves)
    ref = torch.autograd.grad(want.sum(), exact)
    # against differences: along a direction, (f(+h) - f(-h)) / 2h in 64 bits is off by h^2 times the third derivative
    # (h = 1e-4: 1e-8 of it) and 2^-52 |f| / h, far below the gradient's own bound
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i, (a, b, leaf) in enumerate(zip(got, ref, exact)):
        # a density's error moves a gradient by the same relative amount: p is off by (2 tol) p, then the filter's gradient
        # adds 2^-14 of its largest entry; the rows of a token sum over all of its places (at most 3 * 97 terms of f32 sums)
        bound = (4 * tol + 2.0 ** -13 + 291 * 2.0 ** -23) * b.abs().max().item()
        assert (a.double() - b).abs().max().item() <= bound, (i, (a.double() - b).abs().max().item(), bound)
        d = torch.randn(leaf.shape, generator=gen, device="cuda", dtype=torch.float64)
        d /= d.norm()
        moved = []
        with torch.no_grad():
            for s in (1e-4, -1e-4):
                at = [t + s * d if j == i else t for j, t in enumerate(exact)]
                moved.append(_truth(m, y, at[:5], *at[5:])[0].sum())
        along = ((moved[0] - moved[1]) / 2e-4).item()
        assert abs((a.double() * d).sum().item() - along) <= bound * d.abs().sum().item() + 1e-6 * abs(along) + 1e-6


def test_particles_over_observed_tokens_give_the_sequence_density(G):
    """Every particle sees the same tokens, so the run's log marginal likelihood is the sequence's own log-density, with a
    resampling step between the tokens (init, extend, resample through the generative-function interface)."""
    from genjax_amd import gen, linear_categorical, seed
    from genjax_amd.core import const
    from genjax_amd.families.state_space import delta_filter_step
    from genjax_amd.inference import smc

    m, n, time = _Model(seed=1), 64, 6
    y = _sequences(m, 1, time)

    @gen
    def token(state, previous):
        o, new = delta_filter_step(state, *m.inputs(previous))
        linear_categorical(o.flatten(1), m.w, m.b) @ "y"
        return new

    def run():
        p = smc.init(token, (m.state(n), y[0, :1].expand(n)), const(n), {"y": y[0, 1]})
        for t in range(1, time):
            p = smc.resample(p, method="systematic")
            p = smc.extend(p, token, (p.traces.get_retval(), y[0, t:t + 1].expand(n)), {"y": y[0, t + 1]})
        return p

    p = seed(run)(G.key(5))
    want, tol = _truth(m, y, [t.double() for t in m.tables()], m.w.double(), m.b.double())
    # log N and the log-sum-exp of N equal weights: 2^-22 of log N a token besides the density's own bound
    assert abs(float(p.log_marginal_likelihood()) - want.sum().item()) <= time * (tol + 2.0 ** -20)


def test_latent_tokens_resampled_by_index_equal_gathered_states(G):
    """A particle filter over latent tokens, written twice: through the generative-function interface (whose resampling
    gathers every state) and by hand with the ancestors handed to the next step.  Same keys, same tokens, same states."""
    from genjax_amd.families.state_space import delta_filter_step
    from genjax_amd.inference.smc import systematic_resample
    from genjax_amd import backend as B
    from genjax_amd import seed

    m, n, time = _Model(vocab=50, kheads=2, heads=4, dk=32, dv=20, seed=2), 257, 9
    read = torch.randn(5, 4 * 20, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") * 0.5
    seen = torch.randint(0, 5, (time,), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda", dtype=torch.int32)

    def run(fused):
        def body():
            state, tok, anc, spare = m.state(n), torch.zeros(n, dtype=torch.int32, device="cuda"), None, None
            history, total = [], torch.zeros((), device="cuda")
            for t in range(time):
                if anc is not None:
                    tok = tok[anc.long()]
                    if not fused:
                        state = state[anc.long()]
                if fused:
                    o, new = delta_filter_step(state, *m.inputs(tok), ancestors=anc, out=spare)
                    state, spare = new, state                          # two buffers in turn
                else:
                    o, state = delta_filter_step(state, *m.inputs(tok))
                rows = o.flatten(1)
                logw = G.linear_categorical.logpdf(seen[t:t + 1], rows, read)          # evidence of another vocabulary
                tok = B.sample_linear_categorical(G.key(100 + t), rows, m.w, m.b)
                total = total + torch.logsumexp(logw, 0)
                anc = systematic_resample(logw, n)
                if t > 0:                                              # (at t = 0 all particles are still the same)
                    assert int(anc.unique().numel()) < n               # some ancestor is taken twice
                history.append((tok, anc, logw))
            return state, history, total
        return seed(body)(G.key(8))

    a, b = run(True), run(False)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    for x, z in zip(a[1], b[1]):
        assert all(torch.equal(u, v) for u, v in zip(x, z))


def test_captured_training_step_replays_and_refuses_leaves_of_a_living_graph(G):
    m = _Model(seed=3)
    y = _sequences(m, 2, 70)
    leaves = [t.clone().requires_grad_(True) for t in (m.w, m.b)]
    o = torch.randn(140, m.heads * m.dv, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    q, k, v, g, beta = (t.clone().requires_grad_(True) for t in m.inputs(y[:, :-1]))

    def step():
        from genjax_amd.families.state_space import delta_filter

        f, _ = delta_filter(q, k, v, g, beta)
        lp = G.linear_categorical.logpdf(y[:, 1:].reshape(-1), f.flatten(2).flatten(0, 1), *leaves)
        return [lp.detach(), *torch.autograd.grad(lp, [q, k, v, g, beta, *leaves], torch.ones_like(lp))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for turn in range(4):
        with torch.no_grad():
            v.copy_(torch.randn(v.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(turn)))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))

    # a graph of the same leaves that still lives on the current stream: its capture on another stream is refused
    x = o.clone().requires_grad_(True)
    alive = G.linear_categorical.logpdf(y[:, 1:].reshape(-1), x, m.w, m.b)
    refused = torch.cuda.CUDAGraph()
    with pytest.raises(G.GjxError, match="still lives"):
        with torch.cuda.graph(refused, stream=side):
            static = torch.zeros(4, device="cuda")
            static.add_(1.0)
            G.linear_categorical.logpdf(y[:, 1:].reshape(-1), x, m.w, m.b)
    torch.cuda.synchronize()
    (dx,) = torch.autograd.grad(alive, x, torch.ones_like(alive))       # the eager graph is as good as before
    assert torch.isfinite(dx).all()


def test_second_derivatives_are_refused(G):
    from genjax_amd.families.state_space import delta_filter

    m = _Model()
    y = _sequences(m, 1, 5)
    tables = [t.clone().requires_grad_(True) for t in m.inputs(y[:, :-1])]
    o, _ = delta_filter(*tables)
    with pytest.raises(G.GjxError, match="differentiated again"):
        torch.autograd.grad(o.sum(), tables, create_graph=True)
    w = m.w.clone().requires_grad_(True)
    lp = G.linear_categorical.logpdf(y[0, 1:], o.detach().flatten(2)[0], w)
    with pytest.raises(G.GjxError, match="differentiated again"):
        torch.autograd.grad(lp.sum(), w, create_graph=True)


def test_shapes_that_linear_categorical_refuses(G):
    x, w = torch.zeros(3, 8, device="cuda"), torch.zeros(5, 8, device="cuda")
    y = torch.zeros(3, dtype=torch.int32, device="cuda")
    for args, message in (((y, x[None], w), "must be"), ((y[:, None], x, w), "one value or one per row"), ((y[:2], x, w), "against")):
        with pytest.raises(G.GjxError, match=message):
            G.linear_categorical.logpdf(*args)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_padding_is_not_read_by_the_gradient(G, dtype):
    """Whatever stands behind a sequence's length (NaN here, in the inputs and in the upstream gradient) changes nothing:
    the gradients are those of the clean batch, bit for bit, and 0 at the padding."""
    from genjax_amd.families.state_space import delta_filter

    t = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    m = _Model(kheads=1, heads=2, dk=48, dv=40)
    lengths = torch.tensor([0, 1, 64, 100, 130], dtype=torch.int32, device="cuda")
    y = _sequences(m, 5, 130)
    clean = [a.to(t) if i < 3 else a for i, a in enumerate(m.inputs(y[:, :-1]))]
    d_o = torch.randn(5, 130, 2, 40, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(t)

    def grads(args, up):
        leaves = [a.detach().clone().requires_grad_(True) for a in args]
        o, s = delta_filter(*leaves, lengths=lengths)
        return torch.autograd.grad([o, s], leaves, [up, torch.ones_like(s)])

    want = grads(clean, d_o)
    dirty, up = [a.clone() for a in clean], d_o.clone()
    for i, l in enumerate(lengths.tolist()):
        for a in (*dirty, up):
            a[i, l:] = float("nan")
    got = grads(dirty, up)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
        for i, l in enumerate(lengths.tolist()):
            assert not a[i, l:].any()


def test_step_takes_states_inside_a_buffer_and_refuses_outputs_over_inputs(G):
    from genjax_amd.families.state_space import delta_filter_step

    m = _Model(kheads=1, heads=1, dk=1, dv=1)
    tok = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    buffer = torch.randn(3, 1, 1, 1, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    a = delta_filter_step(buffer[1:], *m.inputs(tok))                   # 4 bytes into its storage
    b = delta_filter_step(buffer[1:].clone(), *m.inputs(tok))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(G.GjxError, match="aligned"):
        delta_filter_step(buffer[1:], *m.inputs(tok), out=buffer[1:])
    q, k, v, g, beta = m.inputs(tok)
    with pytest.raises(G.GjxError, match="must not overlap `v`"):
        delta_filter_step(m.state(2), q, k, v, g, beta, out=v.view(2, 1, 1, 1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_two_graphs_of_a_fit_that_keeps(G, dtype):
    """Captured log-density and gradient over what the forward keeps: two graphs, replayed in turn with eager calls between."""
    from genjax_amd import backend as B

    t = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    sets = []
    for i, (n, vocab, width) in enumerate(((100, 700, 512), (65, 3000, 576))):
        gen = torch.Generator("cuda").manual_seed(i)
        x = torch.randn(n, width, device="cuda", generator=gen).to(t)
        w = (torch.randn(vocab, width, device="cuda", generator=gen) / width ** 0.5).to(t)
        y = torch.randint(0, vocab, (n,), device="cuda", generator=gen, dtype=torch.int32)
        up = torch.ones(n, device="cuda")

        def call(x=x, w=w, y=y, up=up):
            lp, lse, kept = B.linear_categorical_logpdf(y, x, w, keep=True)
            assert kept is not None
            return [lp, lse] + B.linear_categorical_grad(y, x, w, None, lse, up, want=(True, True, False), kept=kept)[:2]

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call()
        sets.append((graph, outs, call, x))
    for turn in range(4):
        for graph, outs, call, x in sets:
            x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(turn)))
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_two_threads_on_streams_of_their_own(G):
    """Training steps of two host threads, each on its own stream, give the bits of the same steps one after the other."""
    import threading

    from genjax_amd.families.state_space import delta_filter

    models = [_Model(seed=4, dk=64, dv=64), _Model(seed=5, vocab=90, kheads=2, heads=2, dk=30, dv=33)]
    data = [_sequences(m, 2, 150, seed=i) for i, m in enumerate(models)]

    def step(m, y):
        leaves = [t.clone().requires_grad_(True) for t in (*m.inputs(y[:, :-1]), m.w, m.b)]
        o, last = delta_filter(*leaves[:5])
        lp = G.linear_categorical.logpdf(y[:, 1:].reshape(-1), o.flatten(2).flatten(0, 1), *leaves[5:])
        return [lp.detach(), last.detach(), *torch.autograd.grad(lp, leaves, torch.ones_like(lp))]

    want = [step(m, y) for m, y in zip(models, data)]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[i] = step(models[i], data[i])
            stream.synchronize()
        except BaseException as e:                               # noqa: BLE001  reported below, on the test's thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_longest_rows_and_widest_states(G):
    """The documented ends of the ranges: width 65536, one value in the vocabulary; dv = 1024 with dk = 128, 1024 heads."""
    from genjax_amd.families.state_space import delta_filter, delta_filter_step

    gen = torch.Generator("cuda").manual_seed(0)
    x, w = (torch.randn(n, 65536, device="cuda", generator=gen) / 256.0 for n in (40, 3))
    y = torch.randint(0, 3, (40,), device="cuda", generator=gen, dtype=torch.int32)
    want = torch.log_softmax(x.double() @ w.double().t(), 1).gather(1, y.long()[:, None]).squeeze(1)
    mag = (x.double().abs() @ w.double().abs().t()).max().item()
    tol = 2 * 2 * 65536 * 2.0 ** -23 * mag + 2.0 ** -16 + 2.0 ** -20          # a chain of 65536 products in f32, twice
    assert ((G.linear_categorical.logpdf(y, x, w) - want).abs() <= tol).all()
    assert torch.equal(G.linear_categorical.logpdf(y, x, w[:1]), torch.zeros(40, device="cuda"))
    for heads, dk, dv in ((1, 128, 1024), (1024, 8, 4)):
        q, k = (torch.nn.functional.normalize(torch.randn(1, 3, heads, dk, device="cuda", generator=gen), dim=-1) for _ in range(2))
        v, g = torch.randn(1, 3, heads, dv, device="cuda", generator=gen), -torch.rand(1, 3, heads, device="cuda", generator=gen)
        beta = torch.rand(1, 3, heads, device="cuda", generator=gen)
        o, last = delta_filter(q, k, v, g, beta)
        state = torch.zeros(1, heads, dk, dv, device="cuda")
        for t in range(3):
            one, state = delta_filter_step(state, *(a[:, t] for a in (q, k, v, g, beta)))
            # each side within 2^-15 of the largest entry (its own tests)
            assert ((one - o[:, t]).abs().max() <= 2.0 ** -14 * o.abs().max()).item()
        assert ((state - last).abs().max() <= 2.0 ** -14 * last.abs().max()).item()


@pytest.mark.parametrize("which", ["row", "step"])
def test_captured_calls_refuse_leaves_behind_the_entry_points_own_operations(G, which):
    """As above, where the entry point itself broadcasts the leaf (a shared feature row) or adds an axis to it (one token)."""
    from genjax_amd.families.state_space import delta_filter_step

    m = _Model(kheads=1, heads=1, dk=8, dv=8)
    tok = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    q, k, v, g, beta = m.inputs(tok)
    leaf = (torch.ones(m.w.shape[1], device="cuda") if which == "row" else v.detach().clone()).requires_grad_(True)
    call = (lambda: G.linear_categorical.logpdf(tok, leaf, m.w)) if which == "row" else \
        (lambda: delta_filter_step(m.state(3), q, k, leaf, g, beta)[0])
    alive = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(G.GjxError, match="still lives"):
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            torch.zeros(4, device="cuda").add_(1.0)
            call()
    torch.cuda.synchronize()
    assert torch.isfinite(torch.autograd.grad(alive.sum(), leaf)[0]).all()
