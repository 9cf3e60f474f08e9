"""Plain forms of the training head in 64 bits on the CPU, and how far the kernels may be from them.

u is half a step of float32 (2^-24), h half a step of the result's type.  The bounds count roundings: a sum of k terms, in
whatever order, is off by at most (longest chain of additions) u times the sum of the absolute values."""
import math

import numpy as np
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return float(torch.finfo(dtype).tiny)


# ---- dropout ---------------------------------------------------------------------------------------------------------

def philox_bits(n, seed, offset):
    """16 random bits per element (Philox-4x32-10, eight elements per counter)."""
    m = np.uint64(0xFFFFFFFF)
    blocks = np.arange((n + 7) // 8, dtype=np.uint64)
    c = [blocks & m, blocks >> np.uint64(32), np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, (offset >> 32) & 0xFFFFFFFF)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = np.stack(c, 1).astype("<u4")
    return np.ascontiguousarray(words).view("<u2").reshape(-1)[:n]


def dropout(x, p, seed, offset):
    """Exact: the product is rounded to float32 and then to the type, as documented."""
    below = round(65536 * (1 - p))
    keep = torch.from_numpy(philox_bits(x.numel(), seed % 2 ** 64, offset % 2 ** 64).astype(np.int64) < below).reshape(x.shape)
    factor = np.float32(65536 / below) if below else np.float32(0)
    y = (x.detach().cpu().float() * float(factor)).to(x.dtype)
    return torch.where(keep, y, torch.zeros_like(y)), keep


# ---- layer norm ------------------------------------------------------------------------------------------------------

def layer_norm(x, weight, bias, eps, grad=None):
    """(value, bound) of y and, with grad, of dx, dweight, dbias."""
    kind, d, rows = x.dtype, x.shape[1], x.shape[0]
    wkind = next((t.dtype for t in (weight, bias) if t is not None), torch.float32)   # the type the parameters' gradients are rounded to
    x64 = x.double().cpu()
    w = weight.double().cpu() if weight is not None else torch.ones(d, dtype=torch.float64)
    b = bias.double().cpu() if bias is not None else torch.zeros(d, dtype=torch.float64)
    mean = x64.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x64 - mean) ** 2).mean(1, keepdim=True) + eps)
    hat = (x64 - mean) * rstd
    y = hat * w + b
    # a thread adds at most 32 (wide rows: d / 1024) values, then come 6 exchanges and 16 waves
    chain = 64 + d / 1024
    dmean = chain * U * x64.abs().mean(1, keepdim=True)
    # the mean's error moves every difference alike; the variance and the root add (chain + 8) u of hat, and the mean's error
    # enters the variance to second order only (the differences sum to 0), which one more unit covers
    dhat = dmean * rstd * (1 + dmean * rstd * hat.abs()) + hat.abs() * (chain + 8) * U
    out = [(y, dhat * w.abs() + 3 * U * (y.abs() + (hat * w).abs()) + half_step(kind) * y.abs() + tiny(kind))]
    if grad is not None:
        g64 = grad.double().cpu()
        g = g64 * w
        s0, s1 = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
        dx = rstd * (g - s0 - hat * s1)
        ds0 = chain * U * g.abs().mean(1, keepdim=True)
        ds1 = chain * U * (g * hat).abs().mean(1, keepdim=True) + (g.abs() * dhat).mean(1, keepdim=True)
        size = g.abs() + s0.abs() + (hat * s1).abs()
        e = rstd * (ds0 + hat.abs() * ds1 + dhat * s1.abs() + 6 * U * size) + (chain + 8) * U * dx.abs()
        out.append((dx, e + half_step(kind) * dx.abs() + tiny(kind)))
        # at most rows / 512 rows per block's chain and 32 joins of teams and 32 + 16 of blocks
        rchain = rows / 8 + 128
        dw = (g64 * hat).sum(0)
        e = rchain * U * (g64 * hat).abs().sum(0) + (g64.abs() * dhat).sum(0)
        out.append((dw, e + half_step(wkind) * (dw.abs() + e) + tiny(wkind)))
        db = g64.sum(0)
        e = rchain * U * g64.abs().sum(0)
        out.append((db, e + half_step(wkind) * (db.abs() + e) + tiny(wkind)))
    return out


# ---- softmax loss ----------------------------------------------------------------------------------------------------

def softmax_loss(x, table, target, bias, scale, grad=None):
    """(value, bound) of loss and, with grad, of dx and dtable."""
    kind, d = x.dtype, x.shape[1]
    t = target.cpu().long()
    items, rows = table.shape[0], x.shape[0]
    b = torch.zeros(items, dtype=torch.float64) if bias is None else bias.double().cpu()
    out_of = b <= -1e30
    in_range = (t >= 0) & (t < items)
    at = torch.where(in_range, t, torch.zeros_like(t))
    dead = in_range & out_of[at]
    live = in_range & ~dead
    x64 = torch.where(live[:, None], x.double().cpu(), torch.zeros((), dtype=torch.float64))
    t64 = torch.where(out_of[:, None], torch.zeros((), dtype=torch.float64), table.double().cpu())
    z = scale * (x64 @ t64.T) + torch.where(out_of, torch.zeros_like(b), b)
    masked = z.masked_fill(out_of[None], -math.inf)
    lse = torch.where(live, torch.logsumexp(masked, 1), torch.zeros(rows, dtype=torch.float64))
    mine = z.gather(1, at[:, None])[:, 0]
    loss = torch.where(live, lse - mine, torch.zeros_like(lse))
    loss = torch.where(dead, torch.full_like(loss, math.inf), loss)
    p = torch.exp(masked - lse[:, None]) * live[:, None]
    # a score: d products added one after the other, the planes of a float32 product 2^-23 off, and four roundings after it
    size = abs(scale) * (x64.abs() @ t64.abs().T)
    dz = (2 * (d + 16)) * U * size + 4 * U * (z.abs() + torch.where(out_of, torch.zeros_like(b), b).abs())
    dz = dz.masked_fill(out_of[None], 0)
    # lse: the scores' errors weighted, the sum's chain of additions, exp and log, and its own size four times
    dlse = (p * dz).sum(1) + (items / 16 + 64) * U + 4 * U * lse.abs() + dz.amax(1) * 1e-3
    dmine = dz.gather(1, at[:, None])[:, 0]
    out = [(loss, torch.where(live, dlse + dmine + 2 * U * (lse.abs() + mine.abs()), torch.zeros_like(lse)))]
    if grad is not None:
        g = torch.where(live, grad.double().cpu(), torch.zeros((), dtype=torch.float64))[:, None] * scale
        hit = torch.zeros_like(z)
        hit[torch.arange(rows), at] = live.double()
        q = p - hit
        # relative error of a probability: its exponent's error (score, lse, their difference) and the exponential's
        rel = dz + dlse[:, None] + 4 * U * (z.abs() + lse.abs()[:, None]) + 8 * U
        dq = p * rel + 2 * U * (q.abs() + p) + (half_step(kind) * (q.abs() + p * rel) if kind != torch.float32 else 4 * U * q.abs())
        dq = dq.masked_fill(out_of[None], 0)
        # flushed to zero below the smallest normal number
        dq = dq + live.double()[:, None] * 1e-37
        dx = (q * g) @ t64
        e = (dq * g.abs()) @ t64.abs() + (items + 64) * U * (q.abs() * g.abs()) @ t64.abs()
        out.append((dx, e + half_step(kind) * (dx.abs() + e) + 8 * U * dx.abs() + tiny(kind)))
        dt = (q * g).T @ x64
        e = (dq * g.abs()).T @ x64.abs() + (rows + 64) * U * (q.abs() * g.abs()).T @ x64.abs()
        e = e + 4 * U * (q.abs() * g.abs()).T @ x64.abs()
        out.append((dt, e + half_step(kind) * (dt.abs() + e) + tiny(kind)))
    return out


def close(got, want, name=""):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, name
    inf = torch.isinf(value)
    assert torch.equal(got[inf], value[inf]), name
    assert torch.isfinite(got[~inf]).all(), name
    off = (got - value).abs()[~inf]
    limit = bound.expand_as(value)[~inf]
    worst = (off - limit).max() if off.numel() else torch.tensor(-1.0)
    assert worst <= 0, f"{name}: off by {off.max():.3g}, {(off / limit.clamp(min=1e-300)).max():.3g} times the bound"
