"""Plain 64-bit restatements of the latent path (the write, reading back, absorbed
attention over latent pages) on the CPU, one sequence or token at a time.

Bounds, beside request_oracle's.  The RMS norm is fp32 work: a sum of 512 squares (9 adds
a lane, 6 across), a root, a division and two products, under 2^-18 of the value.  Where
several workgroups share a row's tokens, each leaves its share's output rounded to bf16, off
by 2^-8 of it, so by 2^-8 of the share's part of sum_t w_t |v_t|: `pieces`.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from tests import request_oracle as R
from tests.gpu_pool import page_layout
from tests.helpers import bf16_randn

C, PE, W = 512, 64, 576


def exponent(top):
    """The least e >= -126 with top <= 448 2^e, of a number."""
    return max(-126, math.ceil(math.log2(top / 448.0))) if top > 0 else -126


def latents(c, pe, positions, inv_freq, adjacent, factor, weight, eps):
    """([N, 576] fp64 latents, the bound of their fp32 work)."""
    x = c.double()
    work = torch.zeros((len(c), W), dtype=torch.float64)
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
        work[:, :C] = x.abs() * 2.0 ** -18
    k = R.rotate(pe[:, None], positions, inv_freq, None, adjacent, factor)[:, 0]
    a = pe.double().abs() * abs(factor)
    one, two = (slice(0, PE, 2), slice(1, PE, 2)) if adjacent else (slice(0, PE // 2), slice(PE // 2, PE))
    pair = (a[:, one] + a[:, two]) * 2.0 ** -20
    work[:, C:][:, one] = pair
    work[:, C:][:, two] = pair
    return torch.cat([x, k], 1), work


def rows_of(pool, scale, table_row, n, page, block=1):
    """[n, 576] fp64: the first n tokens of a sequence (CPU pools)."""
    t = torch.arange(n)
    pid, off = torch.as_tensor(table_row, dtype=torch.long)[t // page], t % page
    if scale is None:
        return pool[pid, off].double()
    s = scale.view(torch.uint8)[pid, off // block].view(R.E8M0).float().double()
    return pool.view(torch.uint8)[pid, off].view(R.E4M3).float().double() * s[:, None]


def pools(lens, page, bits, block, seed, sigma=1.0):
    """(table, P, (pool, scale) on the CPU), whose slots that no token has are NaN."""
    table, P = page_layout(lens, page, seed)
    x = [bf16_randn((L, W), seed * 7 + b, sigma) for b, L in enumerate(lens)]
    if bits == 16:
        pool, scale = torch.full((P, page, W), math.nan, dtype=torch.bfloat16), None
    else:
        pool = torch.full((P, page, W), 0x7f, dtype=torch.uint8)
        scale = torch.full((P, page // block), 255, dtype=torch.uint8)
    g = torch.Generator().manual_seed(seed)
    for b, L in enumerate(lens):
        for t0 in range(0, L, block):
            t = torch.arange(t0, min(t0 + block, L))
            pid, off = int(table[b, t0 // page]), t % page
            if bits == 16:
                pool[pid, off] = x[b][t]
                continue
            # blocks of very different sizes
            y = x[b][t].double() * 2.0 ** int(torch.randint(-3, 3, (1,), generator=g))
            e = exponent(float(y.abs().max()))
            pool[pid, off] = (y * 2.0 ** -e).float().to(R.E4M3).view(torch.uint8)
            scale[pid, t0 % page // block] = e + 127
    if bits == 16:
        return table, P, (pool, None)
    return table, P, (pool.view(R.E4M3), scale.view(R.E8M0))


def attend(q, rows, visible, scale, pieces):
    """q [n, H, 576] fp64, rows [T, 576] fp64, visible [n] tokens each query sees (a prefix)
    -> (out [n, H, 512], lse [n, H], bound of out, bound of lse), without reading what a query
    does not see."""
    n, H, _ = q.shape
    out, tol_o = torch.zeros((n, H, C), dtype=torch.float64), torch.zeros((n, H, C), dtype=torch.float64)
    lse, tol_l = torch.full((n, H), -math.inf, dtype=torch.float64), torch.zeros((n, H), dtype=torch.float64)
    for i in range(n):
        T = int(visible[i])
        if T <= 0:
            continue
        k = rows[:T]
        s = (q[i] @ k.T) * scale
        z = torch.logsumexp(s, -1)
        w = torch.exp(s - z[:, None])
        size = (q[i].abs() @ k.abs().T).amax(-1) * (W + 8) * 2.0 ** -24
        delta = size * abs(scale)
        out[i], lse[i] = w @ k[:, :C], z
        tol_o[i] = ((1 + pieces) * 2.0 ** -8 + 2.0 ** -12 + 2 * delta)[:, None] * (w @ k[:, :C].abs())
        tol_l[i] = delta + 2.0 ** -18 * (1 + z.abs())
    return out, lse, tol_o, tol_l


def attention(qn, qp, cpu, table, lens, new, page, block, scale, c0=0, pieces=True):
    """attend() for every sequence's new tokens (new None: one row a sequence, which sees
    lens[b] tokens)."""
    pool, sc = cpu
    q = torch.cat([qn, qp], -1).double()
    N, H, _ = q.shape
    res = [torch.zeros((N, H, C), dtype=torch.float64), torch.zeros((N, H), dtype=torch.float64),
           torch.zeros((N, H, C), dtype=torch.float64), torch.zeros((N, H), dtype=torch.float64)]
    at = c0
    for b, L in enumerate(lens):
        n = 1 if new is None else new[b]
        rows = rows_of(pool, sc, table[b], L, page, block)
        vis = [L] if new is None else [max(0, L - n + i + 1) for i in range(n)]
        for r, x in zip(res, attend(q[at:at + n], rows, vis, scale, pieces)):
            r[at:at + n] = x
        at += n
    return res


def gather(cpu, table, start, cu, n, page, block):
    """[n, 576] bf16 with rows outside the ranges 5.0."""
    pool, sc = cpu
    out = torch.full((n, W), 5.0, dtype=torch.bfloat16)
    P, cap = pool.shape[0], table.shape[1] * page
    for b in range(len(table)):
        for r in range(cu[b], min(cu[b + 1], n)):
            t = int(start[b]) + r - cu[b]
            pid = int(table[b, t // page]) if 0 <= t < cap else -1
            if not 0 <= pid < P:
                out[r] = math.nan
                continue
            out[r] = rows_of(pool, sc, np.array([pid]), t % page + 1, page, block)[-1].to(torch.bfloat16)
    return out
