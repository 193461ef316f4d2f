"""Plain 64-bit references of the device-pointer operators, with the error bounds their kernels are held to."""
import math

import torch


def attention(q, k, v, scale, visible, dtype):
    """q [L, H, d], k, v [K, G, d], visible [L, K] bool -> (out, lse, tolerance of out, tolerance of lse), 64-bit.

    Bounds, per output element, with u the half step of `dtype` (finfo.eps / 2),
    p the exact probabilities and A = sum_j p_j |v_j|:
      * probabilities rounded to `dtype`: u A, and below binary16's normal range
        2^-25 per key relative to the row's largest, which is at least 1 before
        the division by l >= 1: K 2^-25 max|v| / l
      * the result rounded to `dtype`: u |out| <= u A, and 2^-25 absolute (subnormal binary16)
      * a score's d products added in 32 bits, no order assumed, each addition
        off by at most one step (2^-23): e = d 2^-23 scale sum|q k|, which
        changes a probability by the factor 1 +- 2e, numerator and sum
      * exponential, running sums over K keys and the joining of parts in 32 bits:
        (K + 64) 2^-23 A
    """
    q, k, v = q.double(), k.double(), v.double()
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    clean = torch.where(visible.any(0)[:, None, None], k, torch.zeros_like(k))
    vclean = torch.where(visible.any(0)[:, None, None], v, torch.zeros_like(v))
    z = torch.einsum("lhd,khd->hlk", q, clean) * scale
    mag = torch.einsum("lhd,khd->hlk", q.abs(), clean.abs()) * abs(scale)
    z = z.masked_fill(~visible[None], -math.inf)
    lse = torch.logsumexp(z, -1) if k.shape[0] else torch.full(z.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    p = torch.exp(z - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
    out = torch.einsum("hlk,khd->lhd", p, vclean)
    a = torch.einsum("hlk,khd->lhd", p, vclean.abs())
    u = torch.finfo(dtype).eps / 2
    keys = visible.sum(-1).double()
    e = (mag.masked_fill(~visible[None], 0.0).amax(-1) if k.shape[0] else torch.zeros_like(lse)) * q.shape[2] * 2.0 ** -23
    rel = (keys[None] + 64) * 2.0 ** -23
    biggest = vclean.abs().amax((0, 2)) if k.shape[0] else torch.zeros(q.shape[1], dtype=torch.float64, device=q.device)
    tol = (2 * u + 2 * e + rel).permute(1, 0)[..., None] * a + 2.0 ** -25
    if dtype == torch.float16:
        tol = tol + (keys * 2.0 ** -25)[:, None, None] * biggest[None, :, None]
    tol_lse = (e + rel).permute(1, 0) + 2.0 ** -22 * (1 + lse.permute(1, 0).abs().nan_to_num(posinf=0.0))
    return out, lse.permute(1, 0), tol, tol_lse


def check(got, want, tol, what):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities differ"
    off = (got - want).abs()[fine]
    if off.numel():
        worst = (off / tol.expand_as(want)[fine]).max().item()
        assert worst <= 1.0, f"{what}: {worst:.3f} times the bound"


def logits(x, history, prompt, repetition, presence, frequency, biases, allowed, dtype):
    """One row in 64 bits -> (values, tolerance).  biases: list of (token, value); allowed: bool [vocab] or None.

    Each of the row's up to six 32-bit operations is off by half a step (2^-24) of
    its own result, none larger than the sum of magnitudes; the result is
    rounded to `dtype` once.
    """
    y = x.double().clone()
    vocab = y.numel()
    mag = y.abs().clone()
    for t in {t for t in history if 0 <= t < vocab}:
        y[t] = y[t] / repetition if y[t] > 0 else y[t] * repetition
        mag[t] = max(mag[t].item(), y[t].abs().item())
    counts = {}
    for t in history[prompt:]:
        if 0 <= t < vocab:
            counts[t] = counts.get(t, 0) + 1
    for t, n in counts.items():
        y[t] -= frequency * n + presence
        mag[t] += abs(frequency) * n + abs(presence)
    for t, b in {t: b for t, b in biases if 0 <= t < vocab}.items():
        y[t] += b
        mag[t] += abs(b)
    if allowed is not None:
        y[~allowed] = -math.inf
    fine = torch.where(torch.isfinite(y), y.abs(), torch.zeros_like(y))
    tol32 = 6 * 2.0 ** -24 * mag.nan_to_num(posinf=0.0)
    return y, tol32, tol32 + (torch.finfo(dtype).eps / 2 * (fine + tol32) + 2.0 ** -25 if dtype != torch.float32 else 0.0)
