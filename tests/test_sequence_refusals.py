"""What the token-sequence operators refuse, before anything reaches a GPU: the Python front end's messages and the C
entry points' status codes (workspace sizes, types, limits).  No GPU needed: every call below returns on the host."""
import ctypes as C

import pytest
import torch


def _B():
    from genjax_amd import backend as B

    return B


def test_linear_categorical_front_end_refusals():
    B = _B()
    x, w, b, y = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(5), torch.zeros(3, dtype=torch.int32)
    bad = [
        ((y, x, torch.zeros(5, 9), b), "must be"),
        ((y, x[0], w, b), "must be"),
        ((y, x, w[:0], b[:0]), "must be"),
        ((y, x, w, torch.zeros(4)), "bias"),
        ((y, x.double(), w.double(), b.double()), "float32 or all bfloat16"),
        ((y, x.half(), w.half(), b.half()), "float32 or all bfloat16"),
        ((y, x.bfloat16(), w, b), "float32 or all bfloat16"),
        ((y, x, w, b), "device tensor"),
    ]
    for args, message in bad:
        with pytest.raises(B.GjxError, match=message):
            B.linear_categorical_logpdf(*args)


def test_linear_categorical_abi_refusals():
    from genjax_amd import _native as N

    L = N.lib()
    p = C.c_void_p(1 << 20)                      # never dereferenced: each call is refused on the host
    size = C.c_int64()

    def code(dtype=0, x=p, x_ld=8, w=p, w_ld=8, n=3, vocab=5, width=8, y=p, lp=p, lse=p, work=p, work_bytes=1 << 30, kept=None,
             kept_bytes=0):
        return L.gjx_linear_categorical_logpdf(dtype, y, x, x_ld, w, w_ld, None, n, vocab, width, lp, lse, kept, kept_bytes, work,
                                               work_bytes, None)

    assert L.gjx_linear_categorical_workspace(0, p, 8, p, 8, 3, 5, 8, 1, C.byref(size)) == 0 and size.value > 0
    assert L.gjx_linear_categorical_workspace(0, p, 8, p, 8, 3, 5, 8, 1, None) == -1
    assert code(dtype=2) == -1 and b"dtype" in L.gjx_last_error()
    assert code(n=-1) == -1 and code(vocab=0) == -1 and code(width=0) == -1
    assert code(x=None) == -1 and code(w=None) == -1 and code(y=None) == -1 and code(lp=None) == -1
    assert code(x_ld=7) == -1 and code(w_ld=7) == -1 and b"stride" in L.gjx_last_error()
    assert code(work=None) == -1 and code(work_bytes=16) == -1 and b"workspace" in L.gjx_last_error()
    assert code(work=C.c_void_p((1 << 20) + 8)) == -1
    assert code(n=(1 << 24) + 1) == -4 and code(vocab=(1 << 24) + 1) == -4
    assert code(width=65537, x_ld=65537, w_ld=65537) == -4
    assert code(n=0, y=None, x=None, w=None, lp=None, lse=None, work=None, work_bytes=0) == 0       # nothing to do
    assert code(n=100, kept=p, kept_bytes=1 << 30) == -1 and b"nothing is kept" in L.gjx_last_error()      # small widths keep nothing
    sizes = dict(n=100, vocab=5, width=256, x_ld=256, w_ld=256)
    assert L.gjx_linear_categorical_workspace(0, p, 256, p, 256, 100, 5, 256, 3, C.byref(size)) == 0 and size.value > 100 * 256 * 4
    assert code(kept=p, kept_bytes=size.value - 1, **sizes) == -1 and b"d_kept" in L.gjx_last_error()
    assert code(kept=C.c_void_p((1 << 20) + 16), kept_bytes=size.value, **sizes) == -1
    for n, vocab, width, dtype in ((33, 1000, 127, 0), (100, 1000, 127, 0), (100, 1000, 511, 1), (1 << 20, 1 << 20, 512, 0)):
        assert L.gjx_linear_categorical_workspace(dtype, p, width, p, width, n, vocab, width, 3, C.byref(size)) == 0 and size.value == 0

    def grad(lse=p, up=p, kept=None, kept_bytes=0, work_bytes=1 << 30):
        return L.gjx_linear_categorical_grad(0, p, p, 8, p, 8, None, 3, 5, 8, lse, up, kept, kept_bytes, p, p, p, p, work_bytes, None)

    assert grad(lse=None) == -1 and grad(up=None) == -1 and grad(work_bytes=16) == -1
    assert grad(kept=p, kept_bytes=1) == -1
    key = (C.c_uint32 * 2)(0, 1)
    assert L.gjx_random_linear_categorical_i32(key, 0, 0, p, 8, p, 8, None, 3, 5, 8, None, p, 1 << 30, None) == -1


def _delta_args(batch=2, time=3, kheads=1, heads=2, dk=8, dv=4, dtype=torch.float32):
    return [torch.zeros(batch, time, kheads, dk, dtype=dtype), torch.zeros(batch, time, kheads, dk, dtype=dtype),
            torch.zeros(batch, time, heads, dv, dtype=dtype), torch.zeros(batch, time, heads), torch.zeros(batch, time, heads)]


DELTA_BAD = [
    (0, lambda t: t[..., 0], "must be"),                                    # q without its last axis
    (1, lambda t: t[:, :2], "must be"),                                     # k shorter than q
    (2, lambda t: t[:1], "must be"),                                        # v of another batch
    (2, lambda t: torch.zeros(2, 3, 0, 4), "multiple"),
    (0, lambda t: None, "`q` must be a tensor"),
    (3, lambda t: t[..., :1], "log_decay"),
    (4, lambda t: t[:, :2], "beta"),
    (0, lambda t: t.double(), "float32 or all bfloat16"),
    (1, lambda t: t.bfloat16(), "float32 or all bfloat16"),
    (2, lambda t: t.half(), "float32 or all bfloat16"),
    (3, lambda t: t.bfloat16(), "must be float32"),
    (4, lambda t: t.double(), "must be float32"),
    (0, lambda t: t, "device tensor"),                                      # good shapes, but host tensors
]


@pytest.mark.parametrize("which,change,message", DELTA_BAD)
def test_delta_filter_front_end_refusals(which, change, message):
    from genjax_amd.families import state_space as S

    B = _B()
    args = _delta_args()
    args[which] = change(args[which])
    with pytest.raises(B.GjxError, match=message):
        S.delta_filter(*args)
    if args[which] is not None and args[which].dim() >= 3:                  # the single-token form, and the same with a gradient
        step = [t[:, 0] for t in args]
        state = torch.zeros(2, 2, 8, 4)
        if message == "beta" or (message == "must be" and which < 2):       # (good single tokens, or a q without its axes)
            return
        with pytest.raises(B.GjxError, match=message):
            S.delta_filter_step(state, *step)
        with pytest.raises(B.GjxError, match=message):
            S.delta_filter_step(state.requires_grad_(True), *step)


def test_delta_filter_sizes_heads_and_options():
    from genjax_amd.families import state_space as S

    B = _B()
    for sizes, message in (({"dk": 129}, "dk = 129"), ({"dv": 1025}, "dv = 1025"), ({"dk": 0}, "dk = 0"), ({"dv": 0}, "dv = 0"),
                           ({"kheads": 2, "heads": 3}, "multiple"), ({"kheads": 2, "heads": 1}, "multiple")):
        with pytest.raises(B.GjxError, match=message):
            S.delta_filter(*_delta_args(**sizes))
    for scale in (torch.tensor(0.5), "0.5", 1j):                             # a tensor would be read at an unknown time
        with pytest.raises(B.GjxError, match="`scale` must be a number"):
            S.delta_filter(*_delta_args(), scale=scale)
        with pytest.raises(B.GjxError, match="`scale` must be a number"):
            S.delta_filter_step(torch.zeros(2, 2, 8, 4), *(t[:, 0] for t in _delta_args()), scale=scale)


def test_delta_filter_step_refusals():
    from genjax_amd.families import state_space as S

    B = _B()
    args = [t[:, 0] for t in _delta_args()]
    state = torch.zeros(2, 2, 8, 4)
    four = [t.unsqueeze(1) for t in args]
    with pytest.raises(B.GjxError, match="axes"):
        S.delta_filter_step(state, *four)
    with pytest.raises(B.GjxError, match="`state` must be"):
        S.delta_filter_step(None, *args)
    for bad in (state[:1], state.double(), state[..., :3], [0.0]):
        with pytest.raises(B.GjxError, match="`state` must be"):
            S.delta_filter_step(bad, *args)
    grad = state.clone().requires_grad_(True)
    with pytest.raises(B.GjxError, match="`out` cannot be given"):
        S.delta_filter_step(grad, *args, out=state)
    with pytest.raises(B.GjxError, match="`state` must be a tensor"):
        S.delta_filter_step(None, args[0].requires_grad_(True), *args[1:])
    args[0].requires_grad_(False)
    for ancestors in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), [0, 1]):
        with pytest.raises(B.GjxError, match="`ancestors` must be int32"):
            S.delta_filter_step(grad, *args, ancestors=ancestors)


def test_spans_of_strided_tensors():
    """What `out` of a step is held against: the bytes from an input's first entry to the end of its last."""
    B = _B()
    q = torch.zeros(2, 1, 8)
    v = torch.zeros(2, 2, 9)[:, :, :4]
    gate = torch.zeros(1, 2).expand(2, 2)
    p = B._delta_step_plan((torch.float32,) * 5, q.shape, q.shape, v.shape, gate.shape, gate.shape, q.stride(), q.stride(), v.stride(),
                           gate.stride(), gate.stride(), None)
    assert p.spans == (64, 64, 4 * (9 * 3 + 4), 8, 8)


def _shape(dtype=0, kheads=1, heads=2, dk=8, dv=4, batch=2, time=3, v_token=8):
    from genjax_amd import _native as N

    three = C.c_int64 * 3
    kv, gate = three(time * kheads * dk, kheads * dk, dk), three(time * heads, heads, 1)
    return N.DeltaShape(dtype, kheads, heads, dk, dv, 0.5, batch, time, kv, kv, three(time * heads * dv, v_token, dv), gate, gate)


def test_delta_filter_abi_refusals():
    from genjax_amd import _native as N

    L = N.lib()
    p = C.c_void_p(1 << 20)                      # never dereferenced: each call is refused on the host
    size = C.c_int64()

    def sizes(shape, keep=0, out=C.byref(size)):
        return L.gjx_delta_filter_workspace(None if shape is None else C.byref(shape), keep, out)

    need = []
    for keep in (0, 1, 2):
        assert sizes(_shape(), keep) == 0 and size.value > 0 and size.value % 256 == 0
        need.append(size.value)
    assert sizes(_shape(), 3) == -1 and sizes(_shape(), -1) == -1 and sizes(_shape(), 0, None) == -1 and sizes(None) == -1
    for bad in (dict(dtype=2), dict(dtype=-1), dict(kheads=0), dict(heads=0), dict(kheads=2, heads=3), dict(batch=-1), dict(time=-1)):
        assert sizes(_shape(**bad)) == -1, bad
    for bad in (dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=1025), dict(batch=(1 << 24) + 1), dict(heads=1025), dict(time=(1 << 30) + 1),
                dict(v_token=(1 << 22) + 1), dict(batch=1 << 20, time=1 << 24)):
        assert sizes(_shape(**bad)) == -4, bad

    def run(shape=None, q=p, g=p, o=p, state=p, keep=0, work=p, work_bytes=1 << 40):
        return L.gjx_delta_filter(C.byref(shape or _shape()), q, p, p, g, p, None, None, o, state, keep, work, work_bytes, None)

    assert run(q=None) == -1 and run(g=None) == -1 and run(o=None) == -1 and run(state=None) == -1
    assert run(work=None) == -1 and run(work_bytes=need[0] - 1) == -1 and run(keep=1, work_bytes=need[1] - 1) == -1
    assert run(work=C.c_void_p((1 << 20) + 128)) == -1 and b"workspace" in L.gjx_last_error()
    assert run(shape=_shape(batch=0), q=None, g=None, o=None, state=None, work=None, work_bytes=0) == 0       # nothing to do

    def grad(do=p, dq=p, kept=p, kept_bytes=1 << 40, work=p, work_bytes=1 << 40):
        return L.gjx_delta_filter_grad(C.byref(_shape()), p, p, p, p, p, None, do, None, dq, p, p, p, p, None, kept, kept_bytes, work,
                                       work_bytes, None)

    assert grad(do=None) == -1 and grad(dq=None) == -1 and grad(kept=None) == -1 and grad(work=None) == -1
    assert grad(kept_bytes=need[1] - 1) == -1 and b"kept" in L.gjx_last_error()
    assert grad(work_bytes=need[2] - 1) == -1 and grad(work=C.c_void_p((1 << 20) + 16)) == -1

    def step(shape, state=p, ancestors=None, o=p, out=C.c_void_p(1 << 21)):
        return L.gjx_delta_filter_step(C.byref(shape), state, ancestors, p, p, p, p, p, o, out, None)

    assert step(_shape()) == -1 and b"time must be 1" in L.gjx_last_error()
    one = _shape(time=1)
    assert step(one, state=None) == -1 and step(one, o=None) == -1 and step(one, out=None) == -1
    assert step(one, ancestors=p, out=p) == -1 and b"ancestors" in L.gjx_last_error()
    assert step(one, state=C.c_void_p((1 << 20) + 4)) == -1 and step(one, out=C.c_void_p((1 << 21) + 8)) == -1
    assert step(_shape(time=1, batch=0), state=None, o=None, out=None) == 0


def test_linear_categorical_far_rows():
    from genjax_amd import _native as N

    L, p, size = N.lib(), C.c_void_p(1 << 20), C.c_int64()
    assert L.gjx_linear_categorical_workspace(0, p, (1 << 22) + 1, p, 8, 3, 5, 8, 0, C.byref(size)) == -4
    assert L.gjx_linear_categorical_workspace(0, p, 8, p, (1 << 22) + 1, 3, 5, 8, 0, C.byref(size)) == -4
    assert L.gjx_linear_categorical_workspace(0, p, 8, p, 8, 3, 5, 8, 4, C.byref(size)) == -1


def _on_host(monkeypatch, stream, capturing):
    """The entry points' autograd side on host tensors: kernels that return zeros, a stream that the test names."""
    from genjax_amd import distributions as D

    B = _B()
    monkeypatch.setattr(B, "_raw_stream", lambda: stream[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(B, "delta_filter", lambda q, k, v, g, beta, state, *rest, **kw: (
        torch.zeros(v.shape), torch.zeros(v.shape[0], v.shape[2], k.shape[3], v.shape[3]), torch.zeros(1)))
    monkeypatch.setattr(B, "linear_categorical_logpdf", lambda y, x, *rest, **kw: (torch.zeros(x.shape[0]), torch.zeros(x.shape[0]), None))
    monkeypatch.setattr(D, "as_col", lambda t: t)
    return B


@pytest.mark.parametrize("which", ["state", "state by ancestors", "v", "row", "rows", "weight", "behind operations"])
def test_captured_calls_find_the_leaves_behind_the_entry_points_own_operations(monkeypatch, which):
    """The one-token form adds the time axis and gathers the states, a shared feature row is broadcast: the leaf stands
    behind them all the same."""
    from genjax_amd import linear_categorical
    from genjax_amd.families import state_space as S

    stream, capturing = [1], [False]
    B = _on_host(monkeypatch, stream, capturing)
    args = [t[:, 0] for t in _delta_args()]
    ancestors = torch.zeros(2, dtype=torch.int32)
    y, w = torch.zeros(3, dtype=torch.int32), torch.zeros(5, 8)
    leaf = {"state": torch.zeros(2, 2, 8, 4), "state by ancestors": torch.zeros(2, 2, 8, 4), "v": args[2].clone(), "row": torch.zeros(8),
            "rows": torch.zeros(3, 8), "weight": w.clone(), "behind operations": torch.zeros(3, 8)}[which].requires_grad_(True)
    calls = {"state": lambda: S.delta_filter_step(leaf, *args)[0],
             "state by ancestors": lambda: S.delta_filter_step(leaf, *args, ancestors=ancestors)[0],
             "v": lambda: S.delta_filter_step(torch.zeros(2, 2, 8, 4), args[0], args[1], leaf, *args[3:])[0],
             "row": lambda: linear_categorical.logpdf(y, leaf, w), "rows": lambda: linear_categorical.logpdf(y, leaf, w),
             "weight": lambda: linear_categorical.logpdf(y, torch.zeros(3, 8), leaf),
             "behind operations": lambda: linear_categorical.logpdf(y, (leaf * 2.0).tanh() + 1.0 if capturing[0] else leaf, w)}
    monkeypatch.setattr(type(y), "is_cuda", property(lambda t: True))
    alive = calls[which]()
    stream[0] = 2
    assert calls[which]() is not None                       # another stream, but no capture: nothing to refuse
    capturing[0] = True
    with pytest.raises(B.GjxError, match="still lives"):
        calls[which]()
    del alive
    assert calls[which]().grad_fn is not None               # its graph is gone


def test_step_refuses_an_output_buffer_that_requires_a_gradient():
    from genjax_amd.families import state_space as S

    B = _B()
    args = [t[:, 0] for t in _delta_args()]
    with pytest.raises(B.GjxError, match="`out` cannot be given"):
        S.delta_filter_step(torch.zeros(2, 2, 8, 4), *args, out=torch.zeros(2, 2, 8, 4, requires_grad=True))


def test_dual_tensors_are_refused():
    """Forward mode: the plain route would return a result without its tangent."""
    from torch.autograd import forward_ad

    import genjax_amd as G
    from genjax_amd.families import state_space as S

    B = _B()
    args, state = _delta_args(), torch.zeros(2, 2, 8, 4)
    x, w, b, y = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(5), torch.zeros(3, dtype=torch.int32)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))        # noqa: E731
        calls = [lambda i=i: S.delta_filter(*(dual(t) if i == j else t for j, t in enumerate(args))) for i in range(5)]
        calls += [lambda: S.delta_filter(*args, initial_state=dual(state)),
                  lambda: S.delta_filter_step(dual(state), *(t[:, 0] for t in args)),
                  lambda: S.delta_filter_step(state, *(dual(t[:, 0]) for t in args)),
                  lambda: G.linear_categorical.logpdf(y, dual(x), w, b), lambda: G.linear_categorical.logpdf(y, x, dual(w), b),
                  lambda: G.linear_categorical.logpdf(y, x, w, dual(b)),
                  lambda: G.normal.logpdf(dual(b), 0.0, 1.0), lambda: G.normal.logpdf(b, dual(b), 1.0),
                  lambda: G.categorical.logpdf(y, dual(x)), lambda: G.multivariate_normal.logpdf(x, dual(x[0]), torch.eye(8))]
        for call in calls:
            with pytest.raises(B.GjxError, match="forward-mode"):
                call()
        with pytest.raises(B.GjxError, match="device tensor"):              # no tangent: as outside
            S.delta_filter(*args)


def test_gradient_entries_check_their_upstream(monkeypatch):
    """An upstream gradient of another shape or type would be read behind its end."""
    B = _B()
    monkeypatch.setattr(B, "_on_current_device", lambda *a: None)
    x, w, y = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int32)
    good = torch.zeros(3)
    for lse, up, name in ((good, torch.zeros(()), "upstream"), (good, torch.zeros(2), "upstream"), (good, torch.zeros(3, 1), "upstream"),
                          (torch.zeros(2), good, "lse"), (good.double(), good, "lse"), (None, good, "lse")):
        with pytest.raises(B.GjxError, match=f"`{name}` must be"):
            B.linear_categorical_grad(y, x, w, None, lse, up)
    args = _delta_args()
    o = torch.zeros(args[2].shape)
    for bad in (o[:1], o[:, :1], o.double(), o.bfloat16(), o.to("meta"), 1.0):
        with pytest.raises(B.GjxError, match="`d_o` must be"):
            B.delta_filter_grad(*args, bad, None, torch.zeros(1, dtype=torch.uint8))
    with pytest.raises(B.GjxError, match="`d_state` must be"):
        B.delta_filter_grad(*args, o, torch.zeros(1, 2, 8, 4), torch.zeros(1, dtype=torch.uint8))


def test_gather_gradient_abi_refusals():
    from genjax_amd import _native as N

    L, p = N.lib(), C.c_void_p(1 << 20)
    run = lambda d=p, s=p, o=p, n=3, row=4, w=p, out=p: L.gjx_gather_states_grad_f32(d, s, o, n, row, w, out, None)      # noqa: E731
    assert run(n=-1) == -1 and run(row=0) == -1
    assert run(d=None) == -1 and run(s=None) == -1 and run(o=None) == -1 and run(w=None) == -1 and run(out=None) == -1
    assert run(n=(1 << 24) + 1) == -4 and run(row=(1 << 30) + 1) == -4 and run(n=1 << 24, row=1 << 20) == -4
    assert run(n=0, d=None, s=None, o=None, w=None, out=None) == 0
