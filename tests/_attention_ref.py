"""Plain 64-bit statements of the attention operators, and how far a kernel's result may be from them.

Tolerances are bounds, element by element.  With u = eps / 2 of the type (a rounding's largest relative error):

* rotation: one rounding of the result, u |x'|, and fp32 arithmetic, three operations on terms of size |a c| + |b s|.
* attention: the result's rounding, u |o|; the weights' rounding before the product with v, u sum_j p_j |v_j|; and the error of
  a weight itself.  A score is a sum of D products in fp32 (each partial sum off by 2^-23 of the sum of magnitudes at most,
  tensor cores truncate), times a constant, through an exponential of relative error 2^-21: a score's error d moves every
  weight by a factor within exp(+-d), numerator and denominator alike, so the output by 2 d sum_j p_j |v_j|.  Sums of
  weights and of products run in fp32: len 2^-23 of the sum of magnitudes each.
"""
import torch


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, cos_sin, positions, interleaved):
    """(rotated [T,H,D] in 64 bits, tolerance)"""
    r = cos_sin.shape[1]
    row = cos_sin.double()[positions.long()]
    c, s = row[:, None, :r // 2], row[:, None, r // 2:]
    y, mag = x.double().clone(), x.double().abs()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    xa, xb = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    mag[..., a] = mag[..., b] = (xa.abs() * c.abs() + xb.abs() * s.abs()).maximum(xb.abs() * c.abs() + xa.abs() * s.abs())
    tol = unit(x.dtype) * y.abs() + 3 * 2.0 ** -24 * mag * (1 + unit(x.dtype)) + torch.finfo(x.dtype).smallest_normal * unit(x.dtype) * 2
    tol[..., r:] = 0
    return y, tol


def attend(q, k, v, scale, allowed):
    """softmax(scale q k^T) v for one head in 64 bits and its tolerance: q [rows, D], k and v [keys, D], allowed [rows, keys].
    What is not allowed does not enter, whatever it holds; a row with nothing allowed is zero."""
    dtype = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    u = unit(dtype)
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    anyone = allowed.any(0)
    k, v = torch.where(anyone[:, None], k, 0), torch.where(anyone[:, None], v, 0)
    scores = (q @ k.T * scale).masked_fill(~allowed, -torch.inf)
    top = scores.amax(1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -torch.inf, 0, top))
    total = p.sum(1, keepdim=True)
    p = torch.where(total > 0, p / torch.where(total > 0, total, 1), 0)
    o, mass = p @ v, p @ v.abs()
    size = (abs(scale) * (q.abs() @ k.abs().T)).masked_fill(~allowed, 0).amax(1, keepdim=True)
    d = q.shape[1] * 2.0 ** -23 * size + 2.0 ** -21 * (1 + size / q.shape[1])
    tol = u * o.abs() + mass * (u * (1 + u) + 2 * d + 2 * k.shape[0] * 2.0 ** -23) + torch.finfo(dtype).smallest_normal
    return o, tol


def decode(q, k_cache, v_cache, page_table, lens, scale=None):
    b, h, d = q.shape
    hk, page = k_cache.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    out, tol = torch.zeros(2, b, h, d, dtype=torch.float64, device=q.device)
    for i, n in enumerate(lens):
        at = torch.arange(n, device=q.device)
        ids = page_table[i].long()[at // page]
        for j in range(hk):
            rows = slice(j * (h // hk), (j + 1) * (h // hk))
            k, v = k_cache[ids, j, at % page], v_cache[ids, j, at % page]
            out[i, rows], tol[i, rows] = attend(q[i, rows], k, v, scale, torch.ones(h // hk, n, dtype=torch.bool, device=q.device))
    return out, tol


def prefill(q, k, v, ends, scale=None):
    """Rows that belong to no sequence are NaN in the result."""
    t, h, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((t, h, d), torch.nan, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for a, b in zip(ends, ends[1:]):
        allowed = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).tril()
        for j in range(h):
            kv = j // (h // k.shape[1])
            out[a:b, j], tol[a:b, j] = attend(q[a:b, j], k[a:b, kv], v[a:b, kv], scale, allowed)
    return out, tol


def assert_close(got, want, tol):
    """Every element within its tolerance; NaN in `want` is not looked at."""
    bad = ~((got.double() - want).abs() <= tol) & ~want.isnan()
    if bad.any():
        at = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off; first at {at}: {got[at].item()} for {want[at].item()}, "
                             f"tolerance {tol[at].item():.3g}")
