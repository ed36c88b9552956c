"""Attention over states of another length in 64 bits on the CPU, and how far a 16-bit result may be
from it.

The bounds count the roundings of the operator's definition (u is half a step of the 16-bit type,
e = 2^-24 half a step of fp32):
  - a score is a sum of dim products in fp32: off by at most (dim + 4) e S, S the sum of the absolute
    products times the scale; its exponential is off by that much relatively, plus 4 e of its own
    exponent's size and 4 e of the exponential itself;
  - a weight is rounded once to the 16-bit type for the product with the values: u relatively (an fp16
    weight below the normal range: 2^-25 absolutely, where the largest weight is at least 1);
  - sums over n states in fp32: n e relatively to the sum of absolute terms;
  - the result is rounded once: u relatively (fp16 below the normal range: 2^-25).
"""
import math

import torch

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the distance of the numbers below the normal range (bf16: nothing)."""
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def taking_part(batch, states, counts=None, mask=None):
    keep = torch.ones((batch, states), dtype=torch.bool)
    if counts is not None:
        keep &= torch.arange(states)[None] < counts.cpu().long()[:, None]
    if mask is not None:
        keep &= mask.cpu() != 0
    return keep


def attention(queries, keys, values, scale, keep, value_step=None):
    """(out, lse, bound of out, bound of lse); queries b x h x q x d, keys and values b x hs x n x d.
    value_step: the relative rounding of a weight before the second product (None: the queries' type)."""
    dtype = queries.dtype
    u, tiny = half_step(dtype), least(dtype)
    up = u if value_step is None else value_step
    share = queries.shape[1] // keys.shape[1]
    gone = ~keep[:, None, :, None]
    q = queries.detach().cpu().double()
    k = keys.detach().cpu().double().masked_fill(gone, 0.0).repeat_interleave(share, 1)
    v = values.detach().cpu().double().masked_fill(gone, 0.0).repeat_interleave(share, 1)
    dim, n = q.shape[3], k.shape[2]
    scores = (q @ k.mT * scale).masked_fill(~keep[:, None, None, :], -math.inf)
    if n == 0:
        top = torch.full(q.shape[:3] + (1,), -math.inf, dtype=torch.float64)
    else:
        top = scores.amax(-1, keepdim=True)
    base = top.masked_fill(top == -math.inf, 0.0)
    weights = torch.exp(scores - base)
    total = weights.sum(-1, keepdim=True)
    some = total.masked_fill(total == 0, 1.0)
    out = weights @ v / some
    lse = (base + total.log()).squeeze(-1)
    # bounds
    sizes = q.abs() @ k.abs().mT * scale
    size = sizes.amax(-1, keepdim=True) if n else torch.zeros_like(top)
    weight_error = E32 * ((dim + 4) * 2 * size + 8 * size / math.log(2) + n + 16)
    absolute = weights @ v.abs() / some
    out_bound = u * out.abs() + (up + weight_error) * absolute * (1 + up) + 2 * tiny
    out_bound = out_bound + tiny * v.abs().sum(2, keepdim=True) / some
    lse_bound = (weight_error + E32 * 4 * (1 + lse[..., None].abs().masked_fill(lse[..., None].isinf(), 0.0))).squeeze(-1)
    return out, lse, 1.01 * out_bound, 1.01 * lse_bound


def check(got, want, bound, what):
    """got is within bound of want.  Where the type of got ends, rounding to nearest gives infinity: fp16's
    largest is 65504 and its next step would end at 65536, so a value of 65520 and more is infinite."""
    if got.dtype == torch.float16:
        bound = bound.expand_as(want)
        over = want.abs() >= 65520
        either = ((want.abs() - 65520).abs() <= bound) & want.isfinite()
        side = torch.where(either, got.detach().cpu().isinf(), over)
        want = torch.where(side, want.sign() * math.inf, want)
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isinf(), want.isinf()), what
    assert not got.isnan().any(), what
    fine = ~want.isinf()
    off = ((got - want).abs() - bound)[fine]
    if off.numel():
        worst = off.argmax()
        assert off[worst] <= 0, (what, float(off[worst]), float(got[fine][worst]), float(want[fine][worst]),
                                 float(bound.expand_as(want)[fine][worst]))


def made(seed, shape, dtype, spread=1.0):
    gen = torch.Generator()
    gen.manual_seed(seed)
    return (torch.randn(shape, generator=gen) * spread).to(dtype)


def gradients(grad_out, queries, keys, values, out, lse, scale, keep):
    """((grad_queries, its bound), (grad_keys, its bound), (grad_values, its bound)) for the out and lse
    that are given.

    As above, and: a derivative of a score is P (dP - delta), dP and delta sums of dim products in fp32
    (off by (dim + 4) e of their absolute sums); it is rounded once to the 16-bit type; the sums over n
    states or m rows are off by n e, m e of their absolute sums."""
    dtype = queries.dtype
    u, tiny = half_step(dtype), least(dtype)
    b, hs, n, dim = keys.shape
    share = queries.shape[1] // hs
    gone = ~keep[:, None, :, None]
    q, g, o = (x.detach().cpu().double() for x in (queries, grad_out, out))
    k = keys.detach().cpu().double().masked_fill(gone, 0.0).repeat_interleave(share, 1)
    v = values.detach().cpu().double().masked_fill(gone, 0.0).repeat_interleave(share, 1)
    lse = lse.detach().cpu().double()[..., None]
    lse = lse.masked_fill(lse == -math.inf, math.inf)
    weights = torch.exp(q @ k.mT * scale - lse).masked_fill(~keep[:, None, None, :], 0.0)
    size = q.abs() @ k.abs().mT * scale
    some = lse.abs().masked_fill(lse.isinf(), 0.0)
    relative = E32 * ((dim + 4) * size + 8 * (size + some) / math.log(2) + 16)
    delta = (g * o).sum(-1, keepdim=True)
    change = g @ v.mT - delta
    change_error = E32 * (dim + 4) * (g.abs() @ v.abs().mT + (g * o).abs().sum(-1, keepdim=True))
    slope = weights * change
    slope_error = weights * (relative * change.abs() + change_error) * (1 + u) + (u + 4 * E32) * slope.abs()
    slope_error = slope_error + tiny * (weights > 0)
    weight_error = weights * (relative * (1 + u) + u) + tiny * (weights > 0)
    rows = queries.shape[2] * share

    def shared(x):
        return x.view(b, hs, share, n, dim).sum(2)

    result = []
    value = slope @ k * scale
    bound = scale * (slope_error @ k.abs() + E32 * (n + 4) * (slope.abs() @ k.abs())) + u * value.abs()
    result.append((value, bound))
    value = shared(slope.mT @ q) * scale
    bound = scale * shared(slope_error.mT @ q.abs() + E32 * (rows + 4) * (slope.abs().mT @ q.abs())) + u * value.abs()
    result.append((value, bound))
    value = shared(weights.mT @ g)
    bound = shared(weight_error.mT @ g.abs() + E32 * (rows + 4) * (weights.mT @ g.abs())) + u * value.abs()
    result.append((value, bound))
    return [(x, 1.02 * y + 2 * tiny) for x, y in result]
