"""The 4-bit row format and the operators on it in 64 bits, written from the definition in include/diffcache_b200.h."""
import math

import torch

GROUP = 32
SCALE_MAX = {torch.bfloat16: 145.0 * 2.0 ** 118, torch.float16: 9352.0}
# a rounding to the type is off by at most half a step, relative to the value
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def quantise(x: torch.Tensor):
    """x (.., D) of a 16-bit type -> (codes, scales) float64 (.., D / 32, 32) and (.., D / 32, 1)."""
    d = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    top = d.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(d).all(-1, keepdim=True)
    s = torch.where(finite, top, torch.zeros_like(top)) / 7.0
    s = s.clamp_max(SCALE_MAX[x.dtype]).to(x.dtype).double()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    c = torch.where(s > 0, torch.where(finite, d, torch.zeros_like(d)) / torch.where(s > 0, s, torch.ones_like(s)),
                    torch.zeros_like(d))
    c = c.round().clamp(-7, 7)          # torch rounds half to even
    return c, torch.where(finite, s, torch.full_like(s, math.nan))


def stored(x: torch.Tensor) -> torch.Tensor:
    """What the rows x stand for once stored: s * c in 64 bits."""
    c, s = quantise(x)
    return (c * s).reshape(x.shape)


def scan(k: torch.Tensor, q: torch.Tensor):
    """k (P, n, D) float64 stored keys, q (P, D) -> dist (P, n) and a bound on what fp32 arithmetic may be off by: every
    product is exact or rounded once (2^-24), D / 16 tensor-core steps and D / 32 scale products add with a relative
    error below 2^-22 of the magnitudes summed, and 65536 - dot is rounded to fp32."""
    dot = (k @ q.double().unsqueeze(-1)).squeeze(-1)
    mag = (k.abs() @ q.double().abs().unsqueeze(-1)).squeeze(-1)
    D = k.shape[-1]
    dist = 65536.0 - dot
    return dist, D * 2.0 ** -22 * mag + dist.abs() * 2.0 ** -23


def attend(q, k, v, mask, scale):
    """q (H, G, D), k / v (H, n, D) float64, mask (H, n) -> out (H, G, D), lse (H, G) in 64 bits, with the tolerances of an
    fp32 computation that rounds `out` to q's type: a logit is off by at most D * 2^-22 of the magnitudes it sums, which
    changes every weight by that factor; n terms are summed in fp32 (n * 2^-23); exp2 and the final division add 2^-20.
    A weight p enters the second product as p s in two bf16 pieces: p = h + x with |x| <= 2^-8 p kept to 2^-8 of itself,
    i.e. 2^-16 of p; p s = round(h s) + y with y = (h s - round(h s)) + x s, at most 2^-8 + 2^-8 of p s, rounded once, i.e.
    2^-15 of p s.  Together 1.5 * 2^-15, below 2^-14."""
    n, D = k.shape[1], k.shape[2]
    x = torch.matmul(q.double(), k.transpose(1, 2)) * scale
    mag = torch.matmul(q.double().abs(), k.abs().transpose(1, 2)) * scale
    dead = ~mask.unsqueeze(1).expand_as(x)
    x = x.masked_fill(dead, -math.inf)
    mag = mag.masked_fill(dead, 0.0)
    empty = ~mask.any(-1)
    p = torch.softmax(x, dim=-1)
    p = torch.where(dead, torch.zeros_like(p), p)
    out = torch.matmul(p, v)
    lse = torch.logsumexp(x, dim=-1)
    out[empty] = 0.0
    lse[empty] = -math.inf
    eps = D * 2.0 ** -22 * (mag.amax(-1) if n else torch.zeros_like(lse))
    spread = torch.matmul(p, v.abs())
    rel = (2.0 * eps + 2.0 ** -14 + n * 2.0 ** -23 + 2.0 ** -20).unsqueeze(-1)
    tol_out = rel * spread + HALF_STEP[q.dtype] * (out.abs() + rel * spread) + 2.0 ** -25
    tol_lse = eps + n * 2.0 ** -23 + 2.0 ** -20 + lse.abs().nan_to_num(posinf=0.0) * 2.0 ** -22
    return out, lse, tol_out, tol_lse


def assert_close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    fin = torch.isfinite(want)
    off = (got - want).abs()[fin] - torch.as_tensor(tol, dtype=torch.float64, device=got.device).expand_as(want)[fin]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {int((off > 0).sum())} values off, worst {float(off.max()):.3e} over"


def bit_equal(got, want):
    """Same values of a 16-bit type, NaN equal to NaN, zeros of either sign equal."""
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7.0).float(), want.nan_to_num(7.0).float())
