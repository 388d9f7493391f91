"""The packed-batch operators in 64 bits (torch, on whatever device the inputs are on), with the
bound that each output element is held to."""
from __future__ import annotations

import math

import torch

# Half a step of a rounding to nearest, relative to the value.
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def attention(q, k, v, first):
    """q [n, H, D], k, v [K, m, D]: row t attends keys 0..first+t.  Returns (out, spread, score),
    all [n, H, D] or [n, H, 1] in 64 bits: the attention, the same sum with |v| (what an error of
    the weights is multiplied with) and sum |q_d k_d| / sqrt(D) of the largest key (what an error of a
    product is relative to)."""
    n, H, D = q.shape
    K, m, _ = k.shape
    q, k, v = (x.double() for x in (q, k, v))
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    spread, score = out.clone(), out[..., :1].clone()
    if m == 0 or n == 0:
        return out, spread, score
    ahead = torch.arange(m, device=q.device)[None] > first + torch.arange(n, device=q.device)[:, None]
    for h in range(H):
        kh, vh = k[h // (H // K)], v[h // (H // K)]
        s = (q[:, h] @ kh.T / math.sqrt(D)).masked_fill(ahead, -math.inf)
        p = torch.softmax(s, -1)
        p = torch.where(ahead.all(-1, keepdim=True), 0.0, p)
        out[:, h], spread[:, h] = p @ vh, p @ vh.abs()
        a = (q[:, h].abs() @ kh.abs().T / math.sqrt(D)).masked_fill(ahead, 0.0)
        score[:, h, 0] = a.amax(-1)
    return out, spread, score


def attention_bound(out, spread, score, io, keys, D):
    """How far a computed element may be from `out`.

    A score is a sum of D products: rounding each product and each partial sum to 32 bits moves it
    by at most (D + 2) 2^-24 sum |q k|, and the conversion to log2 units, the running maximum's
    subtraction and the exponential by another 2^-24 of their arguments (at most 4 x the score's
    size each, counted as 16).  A weight e^s then moves by that much relative to itself, and the
    normalised weights by twice as much.  Sums over the keys add (keys + 16) 2^-24 of the sum of
    |w v|.  With bf16 activations the weights are rounded to bf16 before they meet v, half a step of
    each, once for the product; and the output is rounded to its type."""
    e32 = HALF[torch.float32]
    weight = 2 * (D + 18) * e32 * (score + 1)
    near = spread * (weight + (keys + 16) * e32)
    if io == torch.bfloat16:
        near = near + spread * HALF[torch.bfloat16]
    return near + HALF[io] * out.abs() + 1e-30


def norm_rope(x, w, eps, position, theta, rope_dim):
    """x [n, H, D], w [D] or None, position [n] whole numbers, theta [rope_dim/2] float32.  Returns
    (y, size): the normed and rotated heads, and for every element the size of the pair it was
    rotated from (what an error of the rotation is relative to)."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    size = y.abs().clone()
    if rope_dim:
        angle = (position.to(torch.float32)[:, None] * theta.to(torch.float32)).double()  # float32 by definition
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        a, b = y[..., 0:rope_dim:2].clone(), y[..., 1:rope_dim:2].clone()
        y[..., 0:rope_dim:2], y[..., 1:rope_dim:2] = a * c - b * s, a * s + b * c
        both = a.abs() + b.abs()
        size[..., 0:rope_dim:2] = size[..., 1:rope_dim:2] = both
    return y, size


def norm_rope_bound(y, size, dtype, D):
    """The sum of squares of D values has a relative error of (D + 1) 2^-24, half of which reaches
    its root; the root, the division and two products add 4 roundings, cos and sin half a step each
    and the rotation 2 more; then the output is rounded."""
    e32 = HALF[torch.float32]
    return size * ((D + 1) / 2 + 8) * e32 + HALF[dtype] * y.abs() + 1e-30


# The root mean square error of 32-bit attention against the definition, relative to the output's, stays
# below this.  The bound above is a worst case, some hundred times the error that roundings of random
# sign add up to; bits that a kernel drops would pass it.  A weight's relative error: a score of a few
# units (log2) is rounded some eight times on its way, each by 2^-24 / sqrt(3) of it in the mean, and
# ln(2) of that reaches the weight: 1.5e-7.  Values that have lost all behind their 16th bit are off
# by 2^-17 / sqrt(3) of the power of two above them, 0.75 of that relative to themselves: 3.3e-6, and
# scores from such keys or queries by as much of a standard deviation above one.
RMS32 = 2.0 ** -20


def rms_error(got, want):
    got, want = got.double(), want.double()
    return float((got - want).square().mean().sqrt() / want.square().mean().sqrt())


def two_parts(x):
    """x rounded to the sum of two bf16 values."""
    a = x.to(torch.bfloat16).to(x.dtype)
    return a + (x - a).to(torch.bfloat16).to(x.dtype)
