"""Plain 64-bit restatements of the request-path operators (pages and slots,
rotary positions, 8-bit pages, decode and prompt attention) on the CPU, one
sequence, token or head at a time, and the error bounds the tests hold the
kernels to.

Bounds.  A rounding to a type is off by at most half a step: eps / 2 of the value
(bf16 2^-8, e4m3 2^-4, below e4m3's normal range 2^-10 of the scale).  Attention
adds up w_t v_t with the weights rounded to bf16 once, so an output is off by at
most 2^-8 sum_t w_t |v_t|; its scores are fp32 sums of D products, off by at most
(D + 8) 2^-24 sum_d |q_d k_d| scale =: delta, which moves a weight by 2 delta and
the lse by delta; the fp32 work behind them (exp2, sums, pieces) stays under 2^-12 of
sum_t w_t |v_t| and 2^-18 (1 + |lse|).
"""
from __future__ import annotations

import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu


def extend(table, lens, n_new, stack, free, page, num_pages, n_tokens, base=None):
    """(table, len_out, cu, positions, slots, free_out) of ws_pages_extend."""
    table = np.array(table)
    cap = table.shape[1] * page
    left = min(max(int(free), 0), len(stack))
    top, pre, used, at = left, 0, 0, 0
    len_out, cu = [], [0]
    positions, slots = np.zeros(n_tokens, np.int32), np.full(n_tokens, -1, np.int32)
    for b, (l, n) in enumerate(zip(lens, n_new)):
        l, n = int(l), int(n)
        tokens = max(n, 0)
        fine = l >= 0 and n >= 0 and l + n <= cap
        have = -(-l // page)
        need = -(-(l + n) // page) - have if fine else 0
        ok = fine and at + tokens <= n_tokens and (need == 0 or pre + need <= left)
        if ok:
            for j in range(need):
                table[b, have + j] = stack[top - 1 - (pre + j)]
            if need:
                used = pre + need
            for i in range(n):
                t = l + i
                pid = int(table[b, t // page])
                positions[at + i] = t + (int(base[b]) if base is not None else 0)
                slots[at + i] = pid * page + t % page if 0 <= pid < num_pages else -1
        len_out.append(l + n if ok else -1)
        pre += need
        at += tokens
        cu.append(min(at, n_tokens))
    return table, np.array(len_out, np.int32), np.array(cu, np.int32), positions, slots, left - used


def rotate(x, positions, inv_freq, axis, adjacent, factor=1.0):
    """x [N, H, D] bf16 -> rotated [N, H, D] fp64."""
    x = x.double().clone()
    half = len(inv_freq)
    pos = positions.double().reshape(-1, x.shape[0])
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        ang = pos[axis[i] if axis is not None else 0] * float(inv_freq[i])
        c, s = (ang.cos() * factor)[:, None], (ang.sin() * factor)[:, None]
        u, v = x[:, :, a].clone(), x[:, :, b].clone()
        x[:, :, a], x[:, :, b] = u * c - v * s, v * c + u * s
    return x


def quantise(x):
    """(e4m3 [..., D], e8m0 [...]) of rows x [..., D] by the write's rule."""
    x = x.double()
    top = x.abs().amax(-1)
    e = torch.where(top > 0, torch.ceil(torch.log2(top / 448.0)).clamp(-126, 127),
                    torch.zeros_like(top))
    return (x * torch.exp2(-e)[..., None]).float().to(E4M3), (e + 127).to(torch.uint8).view(E8M0)


def dequantise(x, scale):
    return x.float().double() * scale.float().double()[..., None]


def tokens_of(pool, scale, table_row, kvh, n, page):
    """[n, D] fp64: the first n tokens of a sequence's KV head (CPU pools)."""
    t = torch.arange(n)
    pid, off = torch.as_tensor(table_row, dtype=torch.long)[t // page], t % page
    if scale is None:
        return pool[pid, kvh, off].double()
    x = pool.view(torch.uint8)[pid, kvh, off].view(E4M3)
    return dequantise(x, scale.view(torch.uint8)[pid, kvh, off].view(E8M0))


def attend(q, k, v, visible, scale):
    """One head: q [n, D], k and v [T, D] in fp64, visible [n] tokens each row
    sees (a prefix) -> (out, lse, bound of out, bound of lse), without reading what a
    row does not see."""
    n, D = q.shape
    out, lse = torch.zeros_like(q), torch.full((n,), -math.inf, dtype=torch.float64)
    tol_o, tol_l = torch.zeros_like(q), torch.zeros(n, dtype=torch.float64)
    for i in range(n):
        T = int(visible[i])
        if T <= 0:
            continue
        s = (k[:T] @ q[i]) * scale
        lse[i] = torch.logsumexp(s, 0)
        w = torch.exp(s - lse[i])
        out[i] = w @ v[:T]
        delta = float((k[:T].abs() @ q[i].abs()).max()) * abs(scale) * (D + 8) * 2.0 ** -24
        tol_o[i] = (2.0 ** -8 + 2.0 ** -12 + 2 * delta) * (w @ v[:T].abs())
        tol_l[i] = delta + 2.0 ** -18 * (1 + abs(float(lse[i])))
    return out, lse, tol_o, tol_l


def check(got, want, tol, what):
    """got within tol of want, elementwise; infinities and NaN in the same places."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), \
        f"{what}: infinities in other places"
    fine = torch.isfinite(want)
    over = ((got - want).abs() - tol)[fine]
    if over.numel() and float(over.max()) > 0:
        i = int(over.argmax())
        raise AssertionError(f"{what}: off by {float((got - want).abs()[fine].flatten()[i]):.3g}, "
                             f"allowed {float(tol.expand_as(want)[fine].flatten()[i]):.3g} "
                             f"({int((over > 0).sum())} of {over.numel()})")
