"""The distributions used on the hot path (reference src/genjax/distributions.py:22-25, 51-54,
62-65, 92-95, 159-162, 194-197, 298-301).  Each is a `Distribution` whose sampler draws a whole
column from one Threefry key and whose logpdf is a HIP kernel; the formulas are TFP's
(SURVEY.md section 8a, row a3)."""
from __future__ import annotations

import torch

from . import backend as B
from .core import Distribution, as_col


def _shape_n(shape):
    n = 1
    for s in shape:
        n *= int(s)
    return n


# --------------------------------------------------------------------------- #
# log-densities that autograd can differentiate: generic hmc (mcmc.py:434-578) takes jax.grad of assess();
# here the HIP log-density kernel is the forward and the HIP gradient kernel (gjx_logpdf_grad_f32) the
# backward of a torch.autograd.Function, so that the user's own glue between the sites (a + b * x, ...) is
# differentiated by autograd and the densities by the library.
# --------------------------------------------------------------------------- #
_FORWARD = {"normal": B.normal_logpdf, "uniform": B.uniform_logpdf, "beta": B.beta_logpdf,
            "bernoulli": lambda x, p, _unused: B.bernoulli_logpdf(x, p)}


class _LogpdfFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, kind, x, p1, p2):
        ctx.kind = kind
        ctx.save_for_backward(x, p1, p2)
        return _FORWARD[kind](x, p1, p2)

    @staticmethod
    def backward(ctx, g):
        x, p1, p2 = ctx.saved_tensors
        want = tuple(ctx.needs_input_grad[1:4])
        if ctx.kind == "bernoulli":
            want = (False, want[1], False)
        gx, g1, g2 = B.logpdf_grad(ctx.kind, x, p1, None if ctx.kind == "bernoulli" else p2, g.contiguous(), want=want)
        fit = lambda gr, like: None if gr is None else gr.sum_to_size(like.shape)   # undo the broadcast
        return None, fit(gx, x), fit(g1, p1), fit(g2, p2)


def _logpdf(kind, x, p1, p2=None):
    x, p1 = as_col(x), as_col(p1)
    p2 = as_col(p2) if p2 is not None else torch.zeros((), dtype=torch.float32, device=x.device)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, p1, p2)):
        return _LogpdfFn.apply(kind, x, p1, p2)
    return _FORWARD[kind](x, p1, p2)


# normal(mu, sigma)                                            distributions.py:159-162
normal = Distribution(
    lambda key, shape, mu, sigma: B.sample_normal(key, shape, mu, sigma),
    lambda x, mu, sigma: _logpdf("normal", x, mu, sigma),
    name="normal",
)

# uniform(low, high)                                           distributions.py:194-197
uniform = Distribution(
    lambda key, shape, lo, hi: B.sample_uniform(key, shape, lo, hi),
    lambda x, lo, hi: _logpdf("uniform", x, lo, hi),
    name="uniform",
)

# flip(p) = Bernoulli(probs=p) (bool in the reference; 0.0/1.0 columns here)   distributions.py:51-54
flip = Distribution(
    lambda key, shape, p: B.sample_bernoulli(key, shape, p),
    lambda x, p: _logpdf("bernoulli", x.to(torch.float32), p),
    name="flip",
)


# bernoulli(logits) = Bernoulli(logits=...)                    distributions.py:22-25
# log_prob = -x softplus(-l) - (1 - x) softplus(l) ([3P] TFP), finite for any |l|; sample = uniform < sigmoid(l)
bernoulli = Distribution(
    lambda key, shape, logits: B.sample_bernoulli_logits(key, shape, logits),
    lambda x, logits: B.bernoulli_logits_logpdf(x.to(torch.float32), as_col(logits)),
    name="bernoulli",
)


# beta(a, b)                                                   distributions.py:62-65
# [3P] tfd.Beta samples through a data-dependent gamma rejection sampler whose stream is not reproduced
# (SURVEY.md Appendix C item 4): the draw has the same law (Marsaglia-Tsang gammas on counter-based draws of
# the site key), not the same bits.
beta = Distribution(
    lambda key, shape, a, b: B.sample_beta(key, shape, a, b),
    lambda x, a, b: _logpdf("beta", x, a, b),
    name="beta",
)


# categorical(logits)                                          distributions.py:92-95
class _Categorical(Distribution):
    def _param_event_ndims(self, a):
        return 1

    def sample(self, logits, sample_shape=None, **kwargs):
        from .core import _next_key, batch_size

        logits = as_col(logits)
        key = _next_key()
        if logits.dim() == 2:
            return B.sample_categorical(key, logits)
        n = sample_shape[0] if sample_shape else (batch_size() or 1)
        out = B.sample_categorical(key, logits, n=n)
        return out if (sample_shape or batch_size()) else out[0]


categorical = _Categorical(None, lambda x, logits: B.categorical_logpdf(x, as_col(logits)), name="categorical")


# categorical(logits = x W^T + b) of distributions.py:92-95 without its logits: for vocabularies too large to keep one
# row of them per particle.  The gradient (x, weight, bias) is the library's, as for the densities above.
class _LinearCategoricalFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, weight, bias, keep):
        lp, lse, kept = (*B.linear_categorical_logpdf(y, x, weight, bias, keep=keep), None)[:3]
        ctx.save_for_backward(y, x, weight, bias, lse, kept)
        return lp

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():
            raise B.GjxError("linear_categorical: its gradient cannot be differentiated again (create_graph=True)")
        y, x, weight, bias, lse, kept = ctx.saved_tensors
        return (None, *B.linear_categorical_grad(y, x, weight, bias, lse, g, want=ctx.needs_input_grad[1:4], kept=kept), None)


class _LinearCategorical(Distribution):
    """linear_categorical(x, weight, bias=None): a draw from softmax(x W^T + b) per row.  x: (n, width) rows or one
    (width,) row shared by every particle (sample_shape=(m,): m draws from it); weight: (vocab, width); bias: (vocab,).
    All float32 or all bfloat16 and finite, the bias or -inf (its entry is never drawn and has the log-density -inf);
    sums and log-densities are float32.  Differentiable in x, weight and bias; the forward of a gradient keeps up to 2 GiB
    for it (the exponentials of all logits) until the backward, and what would take more, or many rows of a small width, is
    formed again.  With keep=False nothing is kept: for losses over many calls, whose kept exponentials would add up."""

    def _param_event_ndims(self, a):
        return a.dim() if isinstance(a, torch.Tensor) else 0

    @staticmethod
    def _rows(x, n):
        # (a shared row's gradient is the sum of the n rows', each in x's type: in bfloat16 as many roundings of 2^-8 of a
        # row's gradient, which add up as their signs fall, besides the sum's own)
        if x.dim() not in (1, 2):
            raise B.GjxError(f"linear_categorical: x {tuple(x.shape)} must be (width,) or (n, width)")
        return x if x.dim() == 2 and x.shape[0] == n else x.reshape(-1, x.shape[-1]).expand(n, x.shape[-1])

    def sample(self, x, weight, bias=None, sample_shape=None, **kwargs):
        from .core import _next_key, batch_size

        x, weight, bias = as_col(x), as_col(weight), None if bias is None else as_col(bias)
        if sample_shape and (x.dim() != 1 or len(sample_shape) != 1):
            raise B.GjxError(f"linear_categorical: sample_shape {tuple(sample_shape)} must be one number of draws from one (width,) row "
                             f"(x: {tuple(x.shape)})")
        n = x.shape[0] if x.dim() == 2 else (sample_shape[0] if sample_shape else (batch_size() or 1))
        out = B.sample_linear_categorical(_next_key(), self._rows(x.detach(), n), weight.detach(),
                                          None if bias is None else bias.detach())
        return out if (x.dim() == 2 or sample_shape or batch_size()) else out[0]

    def logpdf(self, y, x, weight, bias=None, keep=True, **kwargs):
        B.no_tangents(self.name, x, weight, bias)
        x, weight, bias = as_col(x), as_col(weight), None if bias is None else as_col(bias)
        y = y if isinstance(y, torch.Tensor) and y.is_cuda else torch.as_tensor(y, device=x.device)
        if y.dim() > 1:
            raise B.GjxError(f"linear_categorical: y {tuple(y.shape)} must be one value or one per row")
        n = x.shape[0] if x.dim() == 2 else y.numel()
        if y.dim() == 1 and x.dim() == 2 and n == 1:
            n = y.numel()
        if y.dim() == 1 and y.numel() not in (1, n):
            raise B.GjxError(f"linear_categorical: {y.numel()} values against {n} rows of x")
        scalar = y.dim() == 0 and x.dim() == 1
        if y.dtype != torch.int32 and weight.dim() == 2:        # outside the vocabulary: the nearest entry, in 64 bits too
            y = y.long().clamp(0, max(weight.shape[0] - 1, 0)).to(torch.int32)
        rows, ys = self._rows(x, n), y
        if ys.shape != (n,):
            ys = ys.reshape(-1).expand(n)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
            out = _LinearCategoricalFn.apply(ys, rows, weight, bias, bool(keep))
            B._note_leaves("linear_categorical", out)
        else:
            out = B.linear_categorical_logpdf(ys, rows, weight, bias, want_lse=False)[0]
        return out.reshape(()) if scalar else out


linear_categorical = _LinearCategorical(None, None, name="linear_categorical")


# multivariate_normal(mu, cov)                                 distributions.py:298-301
class _MvNormal(Distribution):
    def sample(self, mu, cov, **kwargs):
        from .core import _next_key, batch_size

        mu, cov = as_col(mu), as_col(cov)
        n = mu.shape[0] if mu.dim() == 2 else (cov.shape[0] if cov.dim() == 3 else (batch_size() or 1))
        out = B.sample_mvnormal(_next_key(), n, mu, cov)
        return out if (mu.dim() == 2 or cov.dim() == 3 or batch_size()) else out[0]

    def logpdf(self, x, mu, cov, **kwargs):
        B.no_tangents(self.name, x, mu, cov)
        x, mu, cov = as_col(x), as_col(mu), as_col(cov)
        single = x.dim() == 1 and mu.dim() == 1 and cov.dim() == 2
        out = B.mvnormal_logpdf(x.reshape(-1, x.shape[-1]), mu, cov)
        return out[0] if single else out


multivariate_normal = _MvNormal(None, None, name="multivariate_normal")
