"""delta_filter, its gradient and delta_filter_step against the recursion in 64 bits, token by token, on the same inputs.

Tolerances: every product runs in f32-equivalent partial products (2^-23 each at most left out) with f32 sums; the inputs
here keep |k| = 1 and beta < 1, so a step does not enlarge what came before (the map S -> a (I - beta k k^T) S has norm
at most 1) and the roundings of T chunks add up at most linearly: 64 products of 2^-23 a chunk and side, i.e. below
2^-16 of the tensor's largest entry for the up to 4 chunks and sums over up to 128 entries used here, in every f32 result
(2^-14 for the gradients, which pass two such recursions and the sums over dv as well).  A result in bf16 is rounded once more, 2^-8 of the
entry; its own products take two planes (2^-16)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
NAMES = ("q", "k", "v", "log_decay", "beta", "state")


@pytest.fixture(scope="module")
def S():
    from genjax_amd.families import state_space

    assert torch.cuda.is_available()
    return state_space


def _inputs(batch, time, kheads, heads, dk, dv, dtype, seed=0, state=True):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + batch + 31 * time + 101 * heads + dk + dv)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")        # noqa: E731
    unit = lambda t: (t / t.norm(dim=-1, keepdim=True).clamp_min(1e-3)).to(dtype)      # noqa: E731
    a = {"q": unit(r(batch, time, kheads, dk)), "k": unit(r(batch, time, kheads, dk)), "v": r(batch, time, heads, dv).to(dtype),
         "log_decay": -torch.nn.functional.softplus(r(batch, time, heads)) * 0.3, "beta": torch.sigmoid(r(batch, time, heads))}
    a["state"] = r(batch, heads, dk, dv) * 0.3 if state else None
    return a, r(batch, time, heads, dv).to(dtype), r(batch, heads, dk, dv) * 0.2


def _truth(a, lengths=None, scale=None):
    """The recursion one token at a time in 64 bits, differentiable: (o, last state, leaves)."""
    leaf = {n: None if t is None else t.detach().double().requires_grad_(True) for n, t in a.items()}
    q, k, v, g, beta = (leaf[n] for n in NAMES[:5])
    batch, time, heads, dv = v.shape
    dk, group = q.shape[-1], heads // q.shape[2]
    q, k = q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)
    g = g.clamp_min(-100.0)
    mem = torch.zeros(batch, heads, dk, dv, dtype=torch.float64, device="cuda") if leaf["state"] is None else leaf["state"]
    scale = dk ** -0.5 if scale is None else scale
    outs = []
    for t in range(time):
        new = mem * g[:, t].exp()[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (new * k[:, t, :, :, None]).sum(2))
        new = new + k[:, t, :, :, None] * u[:, :, None, :]
        o = scale * (new * q[:, t, :, :, None]).sum(2)
        if lengths is not None:
            on = (lengths > t)[:, None, None]
            new, o = torch.where(on[..., None], new, mem), torch.where(on, o, torch.zeros_like(o))
        mem = new
        outs.append(o)
    o = torch.stack(outs, 1) if outs else torch.zeros(batch, 0, heads, dv, dtype=torch.float64, device="cuda")
    return o, mem, leaf


def _close(name, got, want, eps):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if want.numel() == 0:
        return
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    err, top = (got.double() - want).abs(), want.abs().max().item()
    worst = (err / (eps * top + half * want.abs() + 1e-30)).max().item()
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound (error {err.max().item():.3g}, largest entry {top:.3g})"


def _check(S, a, d_o, d_state, lengths=None, scale=None, grads=True):
    o, last, leaf = _truth(a, lengths, scale)
    args = [a[n] for n in NAMES[:5]]
    got_o, got_s = S.delta_filter(*args, initial_state=a["state"], lengths=lengths, scale=scale)
    assert got_o.dtype == a["v"].dtype and got_s.dtype == torch.float32
    _close("o", got_o, o.detach(), 2.0 ** -15)
    _close("state", got_s, last.detach(), 2.0 ** -16)
    if not grads:
        return
    names = [n for n in NAMES if a[n] is not None]
    mine = {n: a[n].detach().requires_grad_(True) for n in names}
    o2, s2 = S.delta_filter(*(mine[n] for n in NAMES[:5]), initial_state=mine.get("state"), lengths=lengths, scale=scale)
    assert torch.equal(o2.detach(), got_o) and torch.equal(s2.detach(), got_s)
    want = torch.autograd.grad([o, last], [leaf[n] for n in names], [d_o.double(), d_state.double()], allow_unused=True)
    got = torch.autograd.grad([o2, s2], [mine[n] for n in names], [d_o, d_state])
    for n, x, y in zip(names, got, want):
        _close("d" + n, x, torch.zeros_like(leaf[n]) if y is None else y, 2.0 ** -14)


SIZES = [(1, 1, 1, 1, 1, 1), (2, 3, 1, 2, 16, 16), (1, 64, 1, 1, 64, 64), (2, 65, 2, 2, 32, 48), (3, 77, 2, 4, 50, 33),
         (1, 200, 1, 3, 128, 128), (2, 130, 3, 3, 100, 20), (1, 66, 1, 1, 65, 200), (9, 40, 1, 1, 8, 70)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,time,kheads,heads,dk,dv", SIZES)
def test_filter_and_gradients(S, batch, time, kheads, heads, dk, dv, dtype):
    a, d_o, d_state = _inputs(batch, time, kheads, heads, dk, dv, TYPES[dtype])
    _check(S, a, d_o, d_state)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_initial_state_and_own_scale(S, dtype):
    a, d_o, d_state = _inputs(2, 100, 2, 2, 64, 32, TYPES[dtype], state=False)
    _check(S, a, d_o, d_state, scale=0.7)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ragged_lengths(S, dtype):
    time = 150
    a, d_o, d_state = _inputs(7, time, 1, 2, 40, 24, TYPES[dtype])
    lengths = torch.tensor([0, 1, 63, 64, 65, 128, 150], dtype=torch.int32, device="cuda")
    _check(S, a, d_o, d_state, lengths=lengths)
    for n in NAMES[:5]:                                      # what lies behind a sequence is never looked at
        for i, l in enumerate(lengths.tolist()):
            a[n][i, l:] = float("nan")
    o, last = S.delta_filter(*(a[n] for n in NAMES[:5]), initial_state=a["state"], lengths=lengths)
    assert torch.isfinite(o.float()).all() and torch.isfinite(last).all()
    assert torch.equal(last[0], a["state"][0])
    for i, l in enumerate(lengths.tolist()):
        assert torch.equal(o[i, l:], torch.zeros_like(o[i, l:]))
    beyond = torch.full_like(lengths, 10 ** 6)               # lengths behind the end count as the end, negative ones as 0
    b, _, _ = _inputs(7, time, 1, 2, 40, 24, TYPES[dtype])
    full = S.delta_filter(*(b[n] for n in NAMES[:5]), initial_state=b["state"])
    over = S.delta_filter(*(b[n] for n in NAMES[:5]), initial_state=b["state"], lengths=beyond)
    assert torch.equal(full[0], over[0]) and torch.equal(full[1], over[1])
    none = S.delta_filter(*(b[n] for n in NAMES[:5]), initial_state=b["state"], lengths=-beyond)
    assert torch.equal(none[1], b["state"]) and not none[0].any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strided_views_and_broadcast_inputs(S, dtype):
    """q, k, v as slices of one projection, gates with the head axis first, keys shared over the batch."""
    t, batch, time, heads, d = TYPES[dtype], 2, 90, 2, 32
    a, d_o, d_state = _inputs(batch, time, heads, heads, d, d, t)
    fused = torch.cat([a["q"], a["k"], a["v"]], -1).reshape(batch, time, heads, 3 * d)
    a["q"], a["k"], a["v"] = fused[..., :d], fused[..., d:2 * d], fused[..., 2 * d:]
    a["log_decay"] = a["log_decay"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    _check(S, a, d_o, d_state)
    a["q"] = a["q"].permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)       # last axis strided: copied inside
    a["k"] = a["k"][:1].expand(batch, -1, -1, -1)
    a["beta"] = a["beta"][:, :1].expand(-1, time, -1)
    base = {n: a[n] for n in NAMES}
    _check(S, base, d_o, d_state, grads=False)
    k1, b1 = a["k"][:1].detach().clone().requires_grad_(True), a["beta"][:, :1].detach().clone().requires_grad_(True)
    o, last = S.delta_filter(a["q"], k1.expand(batch, -1, -1, -1), a["v"], a["log_decay"], b1.expand(-1, time, -1), initial_state=a["state"])
    got = torch.autograd.grad([o, last], [k1, b1], [d_o, d_state])
    to, ts, leaf = _truth(base)
    want = torch.autograd.grad([to, ts], [leaf["k"], leaf["beta"]], [d_o.double(), d_state.double()])
    _close("dk of a shared key", got[0].double(), want[0].sum(0, keepdim=True), 2.0 ** -6 if t == torch.bfloat16 else 2.0 ** -13)
    _close("dbeta of a shared gain", got[1], want[1].sum(1, keepdim=True), 2.0 ** -11)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_resets_strong_decays_and_extreme_gains(S, dtype):
    """-inf and very negative log-decays forget everything; later tokens of the same chunk keep full accuracy; gains of
    exactly 0 and 1 (their gradients too), a repeated key."""
    a, d_o, d_state = _inputs(2, 140, 1, 1, 32, 16, TYPES[dtype])
    a["log_decay"][:, 10] = -1e4
    a["log_decay"][:, 70] = -float("inf")
    a["log_decay"][0, 71:75] = -90.0
    a["log_decay"][1, 20:40] = 0.0
    a["beta"][:, ::3] = 0.0
    a["beta"][:, 1::3] = 1.0
    a["k"][:, 30:36] = a["k"][:, 30:31]
    _check(S, a, d_o, d_state)
    a["beta"].zero_()                                        # nothing is written: the state only decays
    a["log_decay"].zero_()
    o, last = S.delta_filter(*(a[n] for n in NAMES[:5]), initial_state=a["state"])
    assert torch.equal(last, a["state"])


def test_identical_keys_keep_accuracy(S):
    """The triangular inverse at its worst: 64 equal keys a chunk, gains near 1."""
    a, d_o, d_state = _inputs(1, 128, 1, 1, 16, 16, torch.float32)
    a["k"][:] = a["k"][:, :1]
    a["beta"][:] = 0.999
    a["log_decay"].zero_()
    _check(S, a, d_o, d_state)


def test_empty_time_and_empty_batch(S):
    a, _, _ = _inputs(2, 1, 1, 1, 8, 8, torch.float32)
    z = {n: a[n][:, :0] for n in NAMES[:5]}
    o, last = S.delta_filter(*(z[n] for n in NAMES[:5]), initial_state=a["state"])
    assert o.shape == (2, 0, 1, 8) and torch.equal(last, a["state"])
    st = a["state"].clone().requires_grad_(True)
    o, last = S.delta_filter(*(z[n] for n in NAMES[:5]), initial_state=st)
    assert torch.equal(torch.autograd.grad(last.sum(), st)[0], torch.ones_like(st))
    e = {n: a[n][:0] for n in NAMES}
    o, last = S.delta_filter(*(e[n] for n in NAMES[:5]), initial_state=e["state"])
    assert o.shape == (0, 1, 1, 8) and last.shape == (0, 1, 8, 8)
    o, new = S.delta_filter_step(e["state"], *(e[n][:, 0] for n in NAMES[:5]))
    assert o.shape == (0, 1, 8)


def test_gradient_against_differences(S):
    a, d_o, d_state = _inputs(1, 70, 1, 1, 12, 10, torch.float32)
    leaves = {n: t.clone().requires_grad_(True) for n, t in a.items()}
    f = lambda d: sum((x.double() * y.double()).sum() for x, y in zip(                          # noqa: E731
        S.delta_filter(*(d[n] for n in NAMES[:5]), initial_state=d["state"]), (d_o, d_state)))
    grads = torch.autograd.grad(f(leaves), list(leaves.values()))
    gen = torch.Generator(device="cuda").manual_seed(5)
    for n, g in zip(leaves, grads):
        d = torch.randn(a[n].shape, generator=gen, device="cuda")
        d = d / d.norm()
        h = 2.0 ** -7
        with torch.no_grad():
            num = ((f({**a, n: a[n] + h * d}) - f({**a, n: a[n] - h * d})) / (2 * h)).item()
        ana = (g.double() * d.double()).sum().item()
        # third derivatives of order ten at h^2 / 6 = 2^-16.6, and 2^-16 sums over h: 2^-8 of the gradient's size
        assert abs(num - ana) <= 2.0 ** -7 * max(1.0, g.norm().item()), (n, num, ana)


def test_only_one_output_used_and_partial_gradients(S):
    a, d_o, d_state = _inputs(2, 80, 1, 2, 16, 24, torch.float32)
    o, last, leaf = _truth(a)
    v = a["v"].clone().requires_grad_(True)
    args = [a["q"], a["k"], v, a["log_decay"], a["beta"]]
    got_o, got_s = S.delta_filter(*args, initial_state=a["state"])
    _close("dv from o", torch.autograd.grad(got_o, v, d_o, retain_graph=True)[0],
           torch.autograd.grad(o, leaf["v"], d_o.double(), retain_graph=True)[0], 2.0 ** -14)
    _close("dv from the state", torch.autograd.grad(got_s, v, d_state)[0],
           torch.autograd.grad(last, leaf["v"], d_state.double())[0], 2.0 ** -14)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,kheads,heads,dk,dv", [(1, 1, 1, 1, 1), (3, 1, 2, 16, 16), (5, 2, 4, 50, 33), (7, 1, 1, 64, 64),
                                                  (4, 2, 2, 128, 128), (2, 1, 1, 100, 130), (2, 1, 1, 128, 1024)])
def test_step(S, n, kheads, heads, dk, dv, dtype):
    a, _, _ = _inputs(n, 1, kheads, heads, dk, dv, TYPES[dtype])
    o, last, _ = _truth(a)
    args = [a[x][:, 0] for x in NAMES[:5]]
    got_o, got_s = S.delta_filter_step(a["state"], *args)
    _close("o", got_o, o[:, 0].detach(), 2.0 ** -19)
    _close("state", got_s, last.detach(), 2.0 ** -19)
    anc = torch.randint(0, n, (n,), device="cuda", generator=torch.Generator("cuda").manual_seed(n)).to(torch.int32)
    b = {**a, "state": a["state"][anc.long()]}
    o, last, _ = _truth(b)
    buf = torch.full_like(a["state"], float("nan"))
    got_o, got_s = S.delta_filter_step(a["state"], *args, ancestors=anc, out=buf)
    assert got_s.data_ptr() == buf.data_ptr()
    _close("o after resampling", got_o, o[:, 0].detach(), 2.0 ** -19)
    _close("state after resampling", got_s, last.detach(), 2.0 ** -19)
    st = a["state"].clone()
    o_in, s_in = S.delta_filter_step(st, *args, out=st)                      # in place
    o_out, s_out = S.delta_filter_step(a["state"], *args)
    assert torch.equal(o_in, o_out) and torch.equal(s_in, s_out) and s_in is st
    far = torch.full((n,), 10 ** 9, dtype=torch.int32, device="cuda")       # clamped, never out of range
    _, s_far = S.delta_filter_step(a["state"], *args, ancestors=far)
    _, s_last = S.delta_filter_step(a["state"], *args, ancestors=torch.full_like(far, n - 1))
    assert torch.equal(s_far, s_last)


def test_step_by_step_equals_the_filter_and_its_gradient(S):
    """The serving form against the whole-sequence form, and the step's gradient through ancestors."""
    a, d_o, d_state = _inputs(3, 90, 1, 2, 32, 40, torch.float32)
    o, last = S.delta_filter(*(a[n] for n in NAMES[:5]), initial_state=a["state"])
    st, outs = a["state"], []
    for t in range(90):
        x, st = S.delta_filter_step(st, *(a[n][:, t] for n in NAMES[:5]))
        outs.append(x)
    _close("o", o, torch.stack(outs, 1).double(), 2.0 ** -15)
    _close("state", last, st.double(), 2.0 ** -15)
    anc = torch.tensor([2, 2, 0], dtype=torch.int32, device="cuda")
    leaf = a["state"].clone().requires_grad_(True)
    x, new = S.delta_filter_step(leaf, *(a[n][:, 0] for n in NAMES[:5]), ancestors=anc)
    got = torch.autograd.grad([x, new], leaf, [d_o[:, 0], d_state])[0]
    b = {n: (t[:, :1] if n != "state" else t[anc.long()]) for n, t in a.items()}
    to, ts, tl = _truth(b)
    g = torch.autograd.grad([to, ts], tl["state"], [d_o[:, :1].double(), d_state.double()])[0]
    want = torch.zeros_like(g).index_add_(0, anc.long(), g)
    _close("dstate", got, want, 2.0 ** -14)


def test_streams_graphs_and_same_bits(S):
    from genjax_amd import backend as B

    sets = []
    for batch, time, dtype in ((2, 100, torch.bfloat16), (1, 70, torch.float32)):
        a, d_o, d_state = _inputs(batch, time, 1, 2, 64, 48, dtype)
        args = [a[n] for n in NAMES[:5]]

        def call(a=a, args=args, d_o=d_o, d_state=d_state):
            o, st, kept = B.delta_filter(*args, a["state"], keep=True)
            step = B.delta_filter_step(st, *(t[:, 0] for t in args))
            return [o, st] + B.delta_filter_grad(*args, d_o, d_state, kept) + list(step)

        eager = call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = call()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(eager, other))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call()
        sets.append((graph, outs, call, a))
    for turn in range(4):
        for graph, outs, call, a in sets:
            a["v"].copy_(torch.randn(a["v"].shape, device="cuda", generator=torch.Generator("cuda").manual_seed(turn)))
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(outs, want))


def test_state_beyond_32_bit_offsets(S):
    """n x heads x dk x dv passes 2^31 elements in the one-token form."""
    n, heads, d = 1030, 128, 128
    a, _, _ = _inputs(2, 1, 1, heads, d, d, torch.bfloat16)
    state = torch.zeros(n, heads, d, d, device="cuda")
    state[-2:] = a["state"]
    wide = lambda t: torch.cat([t[:1, 0].expand(n - 2, *t.shape[2:]), t[:, 0]])              # noqa: E731
    o, new = S.delta_filter_step(state, *(wide(a[x]) for x in NAMES[:5]), out=state)
    to, ts, _ = _truth(a)
    _close("o", o[-2:], to[:, 0].detach(), 2.0 ** -19)
    _close("state", new[-2:], ts.detach(), 2.0 ** -19)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("time", [1, 2, 65])
def test_first_decay_of_an_empty_state_has_no_gradient(S, time, dtype):
    """Without an initial state (or with one of zeros) nothing decays at the first token: its gradient is 0, not rounding."""
    a, d_o, d_state = _inputs(3, time, 2, 4, 40, 24, TYPES[dtype], state=False)
    for state in (None, torch.zeros(3, 4, 40, 24, device="cuda")):
        leaves = [a[n].clone().requires_grad_(True) for n in NAMES[:5]]
        o, last = S.delta_filter(*leaves, initial_state=state)
        grads = torch.autograd.grad([o, last], leaves, [d_o, d_state])
        assert not grads[3][:, 0].any() and (time == 1 or grads[3][:, 1].any())
        assert all(g.any() for i, g in enumerate(grads) if i != 3)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("low,high", [(-25.0, -8.0), (-40.0, -39.0), (-9.0, -0.01)])
@pytest.mark.parametrize("time,kheads,heads,dk,dv,state", [(1, 1, 2, 64, 64, True), (65, 1, 2, 32, 48, True), (130, 2, 2, 128, 40, True),
                                                           (70, 1, 1, 50, 33, False)])
def test_gradient_of_strong_decays(S, time, kheads, heads, dk, dv, state, low, high, dtype):
    """dg_t = a_t <G_t, S_{t-1}>, G_t the gradient of the decayed state: each entry is held against its own size,
    a_t |G_t| |S_{t-1}| (Cauchy and Schwarz bound every term of its sums by that), however small the decay is."""
    a, d_o, d_state = _inputs(2, time, kheads, heads, dk, dv, TYPES[dtype], state=state)
    u = torch.rand(2, time, heads, device="cuda", generator=torch.Generator("cuda").manual_seed(time))
    a["log_decay"] = low + (high - low) * u
    leaf = {n: t.detach().double() for n, t in a.items() if t is not None}
    q, k = (leaf[n].repeat_interleave(heads // kheads, 2) for n in "qk")
    mem = leaf.get("state", torch.zeros(2, heads, dk, dv, dtype=torch.float64, device="cuda"))
    before, faded, outs = [], [], []
    for t in range(time):
        before.append(mem)
        new = (mem * leaf["log_decay"][:, t].exp()[..., None, None]).requires_grad_(True)
        faded.append(new)
        w = leaf["beta"][:, t, :, None] * (leaf["v"][:, t] - (new * k[:, t, :, :, None]).sum(2))
        mem = new + k[:, t, :, :, None] * w[:, :, None, :]
        outs.append(dk ** -0.5 * (mem * q[:, t, :, :, None]).sum(2))
    G = torch.autograd.grad([torch.stack(outs, 1), mem], faded, [d_o.double(), d_state.double()])
    decay = leaf["log_decay"].exp()
    before = [b.detach() for b in before]
    want = decay * torch.stack([(g * b).sum((2, 3)) for g, b in zip(G, before)], 1)
    size = decay * torch.stack([g.norm(dim=(2, 3)) * b.norm(dim=(2, 3)) for g, b in zip(G, before)], 1)
    leaves = [a[n].clone().requires_grad_(True) for n in NAMES[:5]]
    o, last = S.delta_filter(*leaves, initial_state=a["state"])
    got = torch.autograd.grad([o, last], leaves, [d_o, d_state])[3]
    worst = ((got.double() - want).abs() / (2.0 ** -14 * size + 2.0 ** -126)).max().item()
    assert worst <= 1.0, f"{worst:.3g} times its bound"


# 320 or 384 tiles of 16 columns: more than the 256 up to which a workgroup of the scans takes one of them
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,time,kheads,heads,dk,dv", [(5, 130, 8, 8, 50, 112), (5, 200, 8, 8, 128, 112), (2, 330, 3, 12, 64, 250),
                                                           (3, 70, 2, 64, 20, 17)])
def test_wide_scans_over_several_chunks(S, batch, time, kheads, heads, dk, dv, dtype):
    assert batch * heads * (-(-dv // 32) * 2) > 256
    a, d_o, d_state = _inputs(batch, time, kheads, heads, dk, dv, TYPES[dtype])
    _check(S, a, d_o, d_state)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_wide_scans_of_ragged_sequences(S, dtype):
    a, d_o, d_state = _inputs(6, 150, 2, 8, 100, 100, TYPES[dtype], state=False)
    lengths = torch.tensor([0, 1, 64, 65, 127, 150], dtype=torch.int32, device="cuda")
    _check(S, a, d_o, d_state, lengths=lengths)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("slow", [False, True])
def test_many_chunks(S, dtype, slow):
    """70 chunks.  What is forgotten within a chunk keeps the bounds of few chunks; with decays of 0.001 a token the
    roundings of all 70 add up, 18 times those of the four chunks that the bounds count (2^-11 and 2^-9)."""
    a, d_o, d_state = _inputs(1, 4485, 1, 2, 64, 32, TYPES[dtype])
    if slow:
        a["log_decay"] = a["log_decay"] * 0.004
    o, last, leaf = _truth(a)
    mine = {n: t.detach().clone().requires_grad_(True) for n, t in a.items()}
    got = S.delta_filter(*(mine[n] for n in NAMES[:5]), initial_state=mine["state"])
    more = 32.0 if slow else 1.0
    _close("o", got[0].detach(), o.detach(), 2.0 ** -15 * more)
    _close("state", got[1].detach(), last.detach(), 2.0 ** -16 * more)
    want = torch.autograd.grad([o, last], [leaf[n] for n in NAMES], [d_o.double(), d_state.double()])
    for n, x, y in zip(NAMES, torch.autograd.grad(got, [mine[n] for n in NAMES], [d_o, d_state]), want):
        _close("d" + n, x, y, 2.0 ** -14 * more)


def test_more_workgroups_than_a_row_of_the_grid(S):
    """2^24 (particle, head) pairs: a launch along one axis would pass 2^32 threads."""
    n, heads = 1 << 20, 16
    gen = torch.Generator("cuda").manual_seed(1)
    q, k, v, g, beta = (torch.rand(*s, device="cuda", generator=gen) for s in [(n, heads, 1)] * 3 + [(n, heads)] * 2)
    state = torch.rand(n, heads, 1, 1, device="cuda", generator=gen)
    o, new = S.delta_filter_step(state, q, k, v, -g, beta)
    faded = state[..., 0, 0].double() * (-g.double()).exp()
    want = faded + k[..., 0] * beta * (v[..., 0] - faded * k[..., 0])
    assert ((new[..., 0, 0] - want).abs() <= 2.0 ** -20).all()                  # a handful of roundings of values below 2
    assert ((o[..., 0] - want * q[..., 0]).abs() <= 2.0 ** -19).all()
    none = [t[:, None, :8][:, :0] for t in (q, k, v, -g, beta)]                 # no token: 2^23 workgroups of 512 threads
    o, new = S.delta_filter(*none, initial_state=state[:, :8])
    assert o.shape == (n, 0, 8, 1) and torch.equal(new, state[:, :8])


def test_step_into_a_buffer_that_a_graph_saved(S):
    """The new state written over a tensor that an autograd graph needs: its backward says so, as for torch's own operations."""
    a, _, _ = _inputs(2, 1, 1, 1, 8, 8, torch.float32)
    args = [a[n][:, 0] for n in NAMES[:5]]
    w = torch.ones_like(a["state"], requires_grad=True)
    for state, out in ((a["state"].clone(), None), (a["state"].clone(), torch.zeros_like(a["state"]))):
        target = state if out is None else out
        y = (w * target).sum()
        S.delta_filter_step(state, *args, out=target)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    y = (w * a["state"]).sum()
    S.delta_filter_step(a["state"], *args)                  # a state that is only read
    y.backward()
    assert torch.equal(w.grad, a["state"])
    with torch.inference_mode():                            # tensors without a version
        plain = a["state"].clone()
        S.delta_filter_step(plain, *args, out=plain)
    assert torch.equal(plain, S.delta_filter_step(a["state"], *args)[1])


@pytest.mark.parametrize("n,shape", [(1, (1, 1, 1)), (5, (2, 3, 5)), (300, (4, 16, 16)), (2000, (1, 1, 2)), (700, (3, 7, 11)), (40, (8, 128, 128)),
                                     (3000, (2, 8, 8))])
def test_gradient_of_gathered_states(S, n, shape):
    """Rows summed by ancestor: spread, sorted, half of them one ancestor's, all of them one's; the same bits every time.
    A sum of c terms in f32, in any order, is off by at most c 2^-24 of the sum of their sizes."""
    from genjax_amd import backend as B

    gen = torch.Generator("cuda").manual_seed(n)
    d = torch.randn(n, *shape, device="cuda", generator=gen)
    spread = torch.randint(0, n, (n,), device="cuda", generator=gen, dtype=torch.int32)
    half = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.5, n // 3, spread).to(torch.int32)
    for anc in (spread, spread.sort()[0], half, torch.full_like(spread, n - 1), torch.arange(n, device="cuda", dtype=torch.int32)):
        want, size = (torch.zeros(n, *shape, device="cuda", dtype=torch.float64).index_add_(0, anc.long(), t.double()) for t in (d, d.abs()))
        got = B.gather_states_grad(d, anc)
        count = torch.bincount(anc.long(), minlength=n).reshape(n, 1, 1, 1)
        assert ((got.double() - want).abs() <= count * 2.0 ** -24 * size).all()
        for _ in range(3):
            assert torch.equal(got, B.gather_states_grad(d, anc))
    far = spread.clone()
    far[0], far[-1] = -7, 10 ** 9                            # taken to the nearest particle, as the forward takes them
    assert torch.equal(B.gather_states_grad(d, far), B.gather_states_grad(d, far.clamp(0, n - 1)))
    odd = torch.empty(d.numel() + 1, device="cuda")[1:].view_as(d).copy_(d)      # not aligned to 16 bytes
    assert ((B.gather_states_grad(odd, half) - B.gather_states_grad(d, half)).abs() <= 2.0 ** -12 * d.abs().max()).all()


def test_gradients_through_repeated_ancestors_have_the_same_bits(S):
    """Eager calls and replays of a captured one, with other ancestors each time."""
    n = 200
    a, d_o, d_state = _inputs(n, 1, 1, 2, 16, 24, torch.float32)
    args = [a[x][:, 0] for x in NAMES[:5]]
    leaf = a["state"].clone().requires_grad_(True)
    gen = torch.Generator("cuda").manual_seed(3)
    anc = torch.randint(0, 9, (n,), device="cuda", generator=gen, dtype=torch.int32)

    def grad():
        o, new = S.delta_filter_step(leaf, *args, ancestors=anc)
        return torch.autograd.grad([o, new], leaf, [d_o[:, 0], d_state])[0]

    first = grad()
    assert all(torch.equal(first, grad()) for _ in range(4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grad()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = grad()
    for turn in range(5):
        anc.copy_(torch.randint(0, 1 + 40 * turn, (n,), device="cuda", generator=gen))
        graph.replay()
        want = grad()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_sequences_beyond_32_bit_offsets(S):
    """v, o and their gradients pass 2^31 entries.  With log-decays of -0.5 nothing reaches further than e^-64 over 128 tokens, so
    the last tokens' outputs are those of the last 192 alone, the first tokens' gradients those of the first 192."""
    time, heads, dk, dv = (1 << 20) + 70, 16, 32, 128
    gen = torch.Generator("cuda").manual_seed(8)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda", dtype=torch.bfloat16)        # noqa: E731
    q, k = (torch.nn.functional.normalize(r(1, time, 1, dk), dim=-1) for _ in range(2))
    v, d_o = r(1, time, heads, dv), r(1, time, heads, dv)
    assert v.numel() > 1 << 31
    g = torch.full((1, 1, 1), -0.5, device="cuda").expand(1, time, heads)
    beta = torch.full((1, 1, 1), 0.5, device="cuda").expand(1, time, heads)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o, last = S.delta_filter(q, k, v, g, beta)
    grads = torch.autograd.grad(o, leaves, d_o)
    first = ((time - 192) // 64) * 64                       # where a chunk begins
    for part, out, gradients in ((slice(first, time), slice(128, None), False), (slice(0, 192), slice(0, 64), True),
                                 (slice(first, time), slice(128, None), True)):
        short = [t.detach()[:, part].clone().requires_grad_(True) for t in leaves]
        o2, s2 = S.delta_filter(*short, g[:, part], beta[:, part])
        if not gradients:
            _close("o", o[:, part][:, out].detach(), o2[:, out].detach().double(), 2.0 ** -14)
            _close("state", last.detach(), s2.detach().double(), 2.0 ** -14)
        else:
            for name, x, y in zip("qkv", grads, torch.autograd.grad(o2, short, d_o[:, part])):
                _close("d" + name, x[:, part][:, out], y[:, out].double(), 2.0 ** -13)
