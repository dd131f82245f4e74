"""The cache-side operators of a request's path, as a user's program calls
them: pages and slots handed out on the GPU, rotary positions with the write
into the pages, decode attention over 8-bit pages, prompt attention.

`own` false: their plain forms, elementary torch operations in 32 bits (angles
in 64).  `own` true: the framework's entry points on the same inputs.

A case is a dict of plain values:
  kind    "pages"   ops.pages_extend (with `done` > 0: ops.pages_release of that
                    many sequences first)
          "rope"    ops.rope_append, or with cache "none" ops.rope
          "decode8" ops.gqa8_decode_full over 8-bit pages
          "prompt"  ops.gqa_prompt
  B, Hkv, G, D, page     sequences, KV heads, query heads per KV head, head width, page size
  new_lo, new_hi         new tokens per sequence, log-uniform
  old_lo, old_hi         tokens per sequence already in the cache, uniform
  cache                  "bf16", "fp8" (e4m3 with a power-of-two scale per token and KV head) or "none"
  rot, axes, pairs       rotary width, position axes, adjacent pairs (else the two halves)
  lens_seed              the lengths' seed (sizes are the case's alone)
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu


def listed():
    return [
        # A decode step's plan: one new token for each of a few users.
        dict(name="pages_b16_step", kind="pages", B=16, page=64, new_lo=1, new_hi=1, old_lo=100,
             old_hi=8000, done=0, lens_seed=1),
        # A serving batch where some requests end and prompts arrive beside single tokens.
        dict(name="pages_b512_mixed", kind="pages", B=512, page=64, new_lo=1, new_hi=2000, old_lo=0,
             old_hi=8000, done=37, lens_seed=2),
        # A decode step's new tokens at the Mixtral-8x7B layer shape.
        dict(name="rope_b32_step", kind="rope", B=32, Hkv=8, G=4, D=128, page=64, new_lo=1, new_hi=1,
             old_lo=500, old_hi=30000, cache="bf16", rot=128, axes=1, pairs=False, lens_seed=3),
        # Prompts of text and images (time, height, width) at the Qwen3-30B-A3B layer shape.
        dict(name="rope_axes_16k", kind="rope", B=4, Hkv=4, G=8, D=128, page=64, new_lo=4000,
             new_hi=4200, old_lo=0, old_hi=0, cache="bf16", rot=128, axes=3, pairs=False, lens_seed=4),
        # Ragged prompts into 8-bit pages, rotary over part of the head, adjacent pairs.
        dict(name="rope_fp8_part", kind="rope", B=13, Hkv=8, G=3, D=96, page=32, new_lo=50,
             new_hi=1500, old_lo=0, old_hi=4000, cache="fp8", rot=64, axes=1, pairs=True, lens_seed=5),
        # One user's decode step over 8-bit pages: launches and the start chain.
        dict(name="kv8_b1_8k", kind="decode8", B=1, Hkv=4, G=8, D=128, page=64, old_lo=8192,
             old_hi=8192, cache="fp8", lens_seed=6),
        # A ragged batch at the Mixtral-8x7B layer shape.
        dict(name="kv8_b16_32k", kind="decode8", B=16, Hkv=8, G=4, D=128, page=64, old_lo=1000,
             old_hi=32000, cache="fp8", lens_seed=7),
        # Many short contexts, narrow heads, an odd group.
        dict(name="kv8_b96_d64", kind="decode8", B=96, Hkv=8, G=5, D=64, page=32, old_lo=1,
             old_hi=4000, cache="fp8", lens_seed=8),
        # One long prompt at the Mixtral-8x7B layer shape.
        dict(name="prompt_b1_8k", kind="prompt", B=1, Hkv=8, G=4, D=128, page=64, new_lo=8192,
             new_hi=8192, old_lo=0, old_hi=0, cache="bf16", lens_seed=9),
        # Chunks of prompts over what is cached of them in 8-bit pages (Qwen3-30B-A3B layer shape).
        dict(name="prompt_chunks_fp8", kind="prompt", B=4, Hkv=4, G=8, D=128, page=64, new_lo=900,
             new_hi=1100, old_lo=500, old_hi=8000, cache="fp8", lens_seed=10),
        # A few drafted tokens each over long contexts.
        dict(name="prompt_draft_5", kind="prompt", B=8, Hkv=8, G=4, D=128, page=64, new_lo=5, new_hi=5,
             old_lo=4000, old_hi=32000, cache="bf16", lens_seed=11),
        # Many short prompts of odd lengths, a width between the powers of two.
        dict(name="prompt_ragged_d96", kind="prompt", B=24, Hkv=8, G=3, D=96, page=32, new_lo=3,
             new_hi=900, old_lo=0, old_hi=300, cache="bf16", lens_seed=12),
    ]


# A drawn case moves and computes at most this (the largest listed cases').
MOST_BYTES = 6.2e8
MOST_FLOPS = 5.4e11
MOST_SCORES = 2.2e9  # scores of a prompt's plain form, padded


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(("pages", "rope", "rope", "decode8", "decode8", "prompt", "prompt", "prompt"))
        c = dict(kind=kind, page=rng.choice((32, 64, 128)), lens_seed=rng.randrange(1 << 30))
        if kind == "pages":
            c.update(B=_log_int(rng, 1, 2000), new_lo=1, new_hi=_log_int(rng, 1, 3000), old_lo=0,
                     old_hi=_log_int(rng, 1, 16000))
            c["done"] = rng.choice((0, 0, c["B"] // 7))
        elif kind == "rope":
            D = rng.choice((64, 80, 96, 128, 128, 128, 160, 256))
            c.update(B=_log_int(rng, 1, 64), Hkv=rng.choice((1, 2, 4, 8)), G=rng.choice((1, 2, 3, 4, 7, 8)),
                     D=D, new_lo=1, new_hi=_log_int(rng, 1, 4000), old_lo=0, old_hi=_log_int(rng, 1, 30000),
                     cache=rng.choice(("none", "bf16", "bf16", "fp8", "fp8")),
                     rot=rng.choice((D, D, D, 16 * max(1, D // 32))), axes=rng.choice((1, 1, 3)),
                     pairs=rng.random() < 0.3)
        elif kind == "decode8":
            top = _log_int(rng, 1, 100000)
            c.update(B=_log_int(rng, 1, 200), Hkv=rng.choice((1, 2, 4, 8)), G=rng.choice((1, 2, 3, 4, 5, 7, 8, 16)),
                     D=rng.choice((64, 96, 128, 128, 128, 160, 192, 256)), old_lo=max(1, top // rng.choice((1, 4, 50))),
                     old_hi=top, cache="fp8")
        else:
            new, old = _log_int(rng, 1, 8000), rng.choice((0, _log_int(rng, 1, 30000)))
            c.update(B=_log_int(rng, 1, 32), Hkv=rng.choice((1, 2, 4, 8)), G=rng.choice((1, 2, 3, 4, 7, 8)),
                     D=rng.choice((64, 96, 128, 128, 128, 192, 256)), new_lo=max(1, new // rng.choice((1, 3, 20))),
                     new_hi=new, old_lo=old // 4, old_hi=old, cache=rng.choice(("bf16", "bf16", "fp8")))
        w = work(c)
        if w["bytes"] > MOST_BYTES or w["flops"] > MOST_FLOPS:
            continue
        old, new = lengths(c)
        if kind == "prompt" and c["B"] * c["Hkv"] * c["G"] * int(new.max()) * int((old + new).max()) > MOST_SCORES:
            continue
        if kind == "decode8" and 2.0 * c["B"] * c["Hkv"] * c["D"] * int(old.max()) > 2e9:
            continue
        return c


# ---------------------------------------------------------------------------
# sizes


def lengths(case):
    """(tokens in the cache before, new tokens) per sequence, of the case alone."""
    r = np.random.RandomState(case["lens_seed"])
    B = case["B"]
    old = r.randint(case["old_lo"], case["old_hi"] + 1, B)
    if "new_lo" not in case:
        return old.astype(np.int64), np.zeros(B, np.int64)
    lo, hi = math.log(case["new_lo"]), math.log(case["new_hi"])
    new = np.rint(np.exp(r.uniform(lo, hi, B))).astype(np.int64)
    new[:case.get("done", 0)] = 0  # requests that end bring nothing
    return old.astype(np.int64), new


def _pages_of(tokens, page):
    return (tokens + page - 1) // page


def work(case):
    old, new = lengths(case)
    page, B = case["page"], case["B"]
    if case["kind"] == "pages":
        done = np.zeros(B, bool)
        done[:case["done"]] = True
        kept = np.where(done, 0, old)
        got = int((_pages_of(kept + new, page) - _pages_of(kept, page)).sum())
        freed = int(_pages_of(old[done], page).sum())
        N = int(new.sum())
        # lengths in and out and new tokens, ids read and written, position and slot
        return {"bytes": 16.0 * B + 8.0 * (got + freed) + 8.0 * N, "flops": 2.0 * N}
    Hkv, G, D = case["Hkv"], case["G"], case["D"]
    Hq, N = Hkv * G, int(new.sum())
    wide = {"bf16": 2 * D, "fp8": D + 1, "none": 0}[case["cache"]]  # a token's K or V of a head
    if case["kind"] == "rope":
        read = N * D * 2 * (Hq + Hkv * (1 if case["cache"] == "none" else 2)) + 4 * N * (case["axes"] + 1)
        wrote = N * Hq * D * 2 + (N * Hkv * D * 2 if case["cache"] == "none" else N * Hkv * 2 * wide)
        return {"bytes": float(read + wrote), "flops": 3.0 * N * (Hq + Hkv) * case["rot"]}
    if case["kind"] == "decode8":
        T = int(old.sum())
        return {"bytes": float(T * Hkv * 2 * wide + B * Hq * (D * 4 + 4)), "flops": 4.0 * T * Hq * D}
    pairs = float((new * old + new * (new + 1) // 2).sum())  # visible (query, key) pairs of a head
    return {"bytes": float(N * Hq * (D * 4 + 4) + (old + new).sum() * Hkv * 2 * wide),
            "flops": 4.0 * pairs * Hq * D}


# ---------------------------------------------------------------------------
# state


def _rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def _randn(shape, g, sigma=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * sigma).to(torch.bfloat16)


def _table(lens, page, spare, perm):
    """A page table that holds `lens` tokens, of shuffled pages, with `spare`
    columns more, and the pages left over."""
    need = _pages_of(lens, page)
    table = np.full((len(lens), int(need.max()) + spare), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += int(n)
    return table, perm[at:]


def prepare(case, seed):
    old, new = lengths(case)
    page, B = case["page"], case["B"]
    r = np.random.RandomState(seed % (1 << 31))
    if case["kind"] == "pages":
        # twice the pages that the old lengths and the new tokens need, at the most
        P = 2 * int(_pages_of(old + new, page).sum()) + B
        spare = int(_pages_of(new, page).max()) + 1
        table, free = _table(old, page, spare, r.permutation(P).astype(np.int32))
        stack = np.full(P, -1, np.int32)
        stack[:len(free)] = free
        done = np.zeros(B, bool)
        done[:case["done"]] = True
        return dict(case=case, P=P, N=int(new.sum()), table=_ints(table), len_in=_ints(old),
                    n_new=_ints(new), stack=_ints(stack), free=_ints([len(free)]),
                    base=_ints(r.randint(0, 5000, B)), done=torch.from_numpy(done).to(DEV))
    g = _rng(seed)
    Hkv, G, D = case["Hkv"], case["G"], case["D"]
    Hq, N, lens = Hkv * G, int(new.sum()), old + new
    P = int(_pages_of(lens, page).sum()) + 3
    table, _ = _table(lens, page, 1, r.permutation(P).astype(np.int32))
    s = dict(case=case, P=P, scale=D ** -0.5, max_len=int(lens.max()), max_new=int(new.max()))
    if case["kind"] == "rope":
        # q, k, v as the fused projection leaves them: rows of one tensor
        qkv = _randn((N, (Hq + 2 * Hkv) * D), g)
        q, k, v = (x.view(N, -1, D) for x in qkv.split((Hq * D, Hkv * D, Hkv * D), 1))
        tok = np.concatenate([np.arange(o, o + n) for o, n in zip(old, new)])
        seq = np.repeat(np.arange(B), new)
        slots = table[seq, tok // page].astype(np.int64) * page + tok % page
        pos = tok[None] + r.randint(0, 100, (1, B))[:, seq]
        if case["axes"] > 1:  # time stands, height and width run over an image of 40 columns
            pos = np.stack([pos[0] // 1200, pos[0] // 40 % 30, pos[0] % 40]) + r.randint(0, 4000, (3, B))[:, seq]
        half = case["rot"] // 2
        inv = torch.from_numpy((1e6 ** (-np.arange(half) / half)).astype(np.float32)).to(DEV)
        axis = [(0 if i % 8 < 3 else 1 + i % 2) for i in range(half)] if case["axes"] > 1 else [0] * half
        s.update(q=q, k=k, v=v, pos=_ints(pos), slots=_ints(slots), inv=inv, axis=axis,
                 axis_dev=torch.tensor(axis, device=DEV))
        if case["cache"] == "bf16":
            s.update(kp=torch.zeros((P, Hkv, page, D), dtype=torch.bfloat16, device=DEV))
            s["vp"] = torch.zeros_like(s["kp"])
        elif case["cache"] == "fp8":
            s.update(kp=torch.zeros((P, Hkv, page, D), dtype=torch.uint8, device=DEV).view(E4M3))
            s["vp"] = torch.zeros((P, Hkv, page, D), dtype=torch.uint8, device=DEV).view(E4M3)
            s["ks"] = torch.full((P, Hkv, page), 127, dtype=torch.uint8, device=DEV).view(E8M0)
            s["vs"] = torch.full((P, Hkv, page), 127, dtype=torch.uint8, device=DEV).view(E8M0)
        return s
    s.update(table=_ints(table), lens=_ints(lens), kp=_randn((P, Hkv, page, D), g), vp=_randn((P, Hkv, page, D), g))
    if case["cache"] == "fp8":  # what the quantised write leaves: a power of two per token and head
        for p, sc in (("kp", "ks"), ("vp", "vs")):
            e = torch.ceil(torch.log2(s[p].float().abs().amax(-1, keepdim=True) / 448.0))
            s[sc] = (e + 127).squeeze(-1).to(torch.uint8).view(E8M0)
            s[p] = (s[p].float() * torch.exp2(-e)).to(E4M3)
    if case["kind"] == "decode8":
        s["q"] = _randn((B, Hq, D), g)
        return s
    s["q"] = _randn((N, Hq, D), g)
    cu = np.concatenate([[0], np.cumsum(new)])
    s["cu"] = _ints(cu)
    # the plain form's padded layout: token of (sequence, i), and whether there is one
    i = np.arange(int(new.max()))[None]
    s["pad"] = torch.from_numpy(np.minimum(cu[:-1, None] + i, N - 1)).to(DEV)
    s["seq"] = torch.from_numpy(np.repeat(np.arange(B), new)).to(DEV)
    s["idx"] = torch.from_numpy(np.concatenate([np.arange(n) for n in new])).to(DEV)
    return s


# ---------------------------------------------------------------------------
# plain forms


def _plain_release(s):
    page, table = s["case"]["page"], s["table"]
    held = torch.where(s["done"], _pages_of(s["len_in"], page), 0).long()
    end = held.cumsum(0)
    col = torch.arange(table.shape[1], device=DEV)
    at = s["free"].long() + (end - held)[:, None] + col  # where a row's pages go
    put = col < held[:, None]
    dump = s["stack"].numel()  # entries that hold no page go behind the stack
    stack = torch.cat([s["stack"], s["stack"].new_zeros(1)])
    stack[torch.where(put, at, dump)] = torch.where(put, table, 0)
    s["stack"].copy_(stack[:dump])
    return torch.where(s["done"], 0, s["len_in"]), (s["free"] + end[-1]).int()


def _plain_extend(s, len_in, free):
    page, table = s["case"]["page"], s["table"]
    n, cap = s["n_new"], page * table.shape[1]
    have = _pages_of(len_in, page)
    fine = (len_in >= 0) & (n >= 0) & (len_in.long() + n <= cap)
    need = torch.where(fine, _pages_of(len_in + n, page) - have, 0).long()
    pre = need.cumsum(0)
    ok = fine & ((need == 0) | (pre <= free))
    first = free - 1 - (pre - need)  # stack place of a sequence's first new page
    col = torch.arange(table.shape[1], device=DEV)
    fresh = ok[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    at = (first[:, None] - (col - have[:, None])).clamp(0, s["stack"].numel() - 1)
    table.copy_(torch.where(fresh, s["stack"][at], table))
    end = n.clamp(min=0).cumsum(0)
    cu = torch.cat([end.new_zeros(1), end])
    t = torch.arange(s["N"], device=DEV)
    b = torch.searchsorted(end, t, right=True)
    held = b < len(n)
    b = b.clamp(max=len(n) - 1)
    pos = len_in[b] + t - cu[b]
    good = held & ok[b]
    pid = table[b, (pos // page).clamp(0, table.shape[1] - 1)]
    slots = torch.where(good & (pid >= 0) & (pid < s["P"]), pid * page + pos % page, -1)
    positions = torch.where(good, pos + s["base"][b], 0)
    used = torch.where(ok, pre, 0).max()
    return (table, torch.where(ok, len_in + n, -1).int(), cu.int(), positions.int(), slots.int(),
            (free - used).int())


def _plain_rotate(x, cos, sin, rot, pairs):
    x = x.float()
    a, rest = x[..., :rot], x[..., rot:]
    if pairs:
        p, q = a[..., 0::2], a[..., 1::2]
        a = torch.stack([p * cos - q * sin, q * cos + p * sin], -1).flatten(-2)
    else:
        p, q = a[..., :rot // 2], a[..., rot // 2:]
        a = torch.cat([p * cos - q * sin, q * cos + p * sin], -1)
    return torch.cat([a, rest], -1)


def _plain_put(pool, scales, slots, x, page):
    """x [N, Hkv, D] in 32 bits into the slots of a pool."""
    pid, off = slots // page, slots % page
    if scales is None:
        pool[pid, :, off] = x.to(torch.bfloat16)
        return
    m, e = torch.frexp(x.abs().amax(-1) / 448.0)  # m 2^e, 1/2 <= m < 1
    e = torch.where(m == 0.5, e - 1, e).clamp(-126, 127)
    scales.view(torch.uint8)[pid, :, off] = (e + 127).to(torch.uint8)
    pool.view(torch.uint8)[pid, :, off] = torch.ldexp(x, -e[..., None]).to(E4M3).view(torch.uint8)


def _plain_rope(s):
    c = s["case"]
    turn = s["pos"].double()[s["axis_dev"]].T * s["inv"].double()  # [N, pairs]
    cos, sin = turn.cos().float()[:, None], turn.sin().float()[:, None]
    q = _plain_rotate(s["q"], cos, sin, c["rot"], c["pairs"]).to(torch.bfloat16)
    k = _plain_rotate(s["k"], cos, sin, c["rot"], c["pairs"])
    if c["cache"] == "none":
        return q, k.to(torch.bfloat16)
    slots = s["slots"].long()
    _plain_put(s["kp"], s.get("ks"), slots, k, c["page"])
    _plain_put(s["vp"], s.get("vs"), slots, s["v"].float(), c["page"])
    return _rope_out(s, q)


def _rope_out(s, q):
    return (q, s["kp"], s["vp"]) + ((s["ks"], s["vs"]) if "ks" in s else ())


def _plain_rows(pool, scales, table):
    """[B, Hkv, tokens, D] in 32 bits, the pages of a table side by side."""
    at = table.long().clamp(min=0)
    if scales is None:
        x = pool[at].float()
    else:
        x = pool.view(torch.uint8)[at].view(E4M3).float()
        x = x * scales.view(torch.uint8)[at].view(E8M0).float()[..., None]
    B, _, Hkv, _, D = x.shape
    return x.transpose(1, 2).reshape(B, Hkv, -1, D)


def _plain_attend(q, k, v, seen, scale):
    """q [B, Hkv, R, D], k and v [B, Hkv, T, D], seen broadcast to [B, Hkv, R, T] ->
    (out, lse) in 32 bits."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous())
    s = s.mul_(scale).masked_fill_(~seen, -torch.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total, (m + total.log()).squeeze(-1)


def _plain_decode8(s):
    B, Hq, D = s["q"].shape
    k, v = (_plain_rows(s[p], s[sc], s["table"]) for p, sc in (("kp", "ks"), ("vp", "vs")))
    seen = torch.arange(k.shape[2], device=DEV) < s["lens"][:, None, None, None]
    out, lse = _plain_attend(s["q"].float().view(B, k.shape[1], -1, D), k, v, seen, s["scale"])
    return out.reshape(B, Hq, D).to(torch.bfloat16), lse.reshape(B, Hq)


def _plain_prompt(s):
    c = s["case"]
    Hkv, G, D = c["Hkv"], c["G"], c["D"]
    k, v = (_plain_rows(s[p], s.get(sc), s["table"]) for p, sc in (("kp", "ks"), ("vp", "vs")))
    B, n = s["pad"].shape
    q = s["q"][s["pad"]].float().view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    new = s["cu"][1:] - s["cu"][:-1]
    at = (s["lens"] - new)[:, None] + torch.arange(n, device=DEV)  # position of query i
    seen = torch.arange(k.shape[2], device=DEV) <= at[..., None]
    out, lse = _plain_attend(q, k, v, seen[:, None].repeat(1, 1, G, 1), s["scale"])
    out = out.view(B, Hkv, G, n, D)[s["seq"], :, :, s["idx"]]
    lse = lse.view(B, Hkv, G, n)[s["seq"], :, :, s["idx"]]
    return out.reshape(-1, Hkv * G, D).to(torch.bfloat16), lse.reshape(-1, Hkv * G)


# ---------------------------------------------------------------------------
# the calls


def _own_run(s):
    from scope_amd import ops

    c = s["case"]
    if c["kind"] == "pages":
        len_in, free = s["len_in"], s["free"]
        if c["done"]:
            len_in, free = ops.pages_release(s["table"], len_in, s["done"], s["stack"], free, c["page"])
        st = ops.pages_extend(s["table"], len_in, s["n_new"], s["stack"], free, c["page"], s["P"], s["N"],
                              pos_base=s["base"])
        return s["table"], st.len_out, st.cu_new, st.positions, st.slots, st.free_out
    if c["kind"] == "rope":
        how = dict(pair_axis=s["axis"], adjacent=c["pairs"])
        if c["cache"] == "none":
            return ops.rope(s["q"], s["k"], s["pos"], s["inv"], **how)
        q = ops.rope_append(s["q"], s["k"], s["v"], s["pos"], s["inv"], s["slots"], s["kp"], s["vp"],
                            k_scale=s.get("ks"), v_scale=s.get("vs"), **how)
        return _rope_out(s, q)
    if c["kind"] == "decode8":
        return ops.gqa8_decode_full(s["q"], s["kp"], s["vp"], s["ks"], s["vs"], s["table"], s["lens"],
                                    s["scale"], s["max_len"])
    return ops.gqa_prompt(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"], s["scale"], s["max_len"],
                          k_scale=s.get("ks"), v_scale=s.get("vs"))


def run(s):
    if own:
        return _own_run(s)
    kind = s["case"]["kind"]
    if kind == "pages":
        len_in, free = s["len_in"], s["free"]
        if s["case"]["done"]:
            len_in, free = _plain_release(s)
        return _plain_extend(s, len_in, free)
    return {"rope": _plain_rope, "decode8": _plain_decode8, "prompt": _plain_prompt}[kind](s)


# ---------------------------------------------------------------------------
# 64 bits, from the definitions, one sequence and KV head at a time


def _token_rows(s, b, h, n, which):
    """[n, D] of sequence b's first n tokens of KV head h, in 64 bits."""
    page = s["case"]["page"]
    t = torch.arange(n, device=DEV)
    pid, off = s["table"][b].long()[t // page], t % page
    pool, sc = {"k": ("kp", "ks"), "v": ("vp", "vs")}[which]
    if sc not in s:
        return s[pool][pid, h, off].double()
    x = s[pool].view(torch.uint8)[pid, h, off].view(E4M3).double()
    e = s[sc].view(torch.uint8)[pid, h, off].double() - 127
    return x * torch.exp2(e)[:, None]


def _exact_attention(s, old, new):
    c = s["case"]
    Hkv, G, D = c["Hkv"], c["G"], c["D"]
    q = s["q"].double().view(-1, Hkv, G, D)
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:-1], dtype=torch.float64, device=DEV)
    row = 0
    for b in range(c["B"]):
        n = int(new[b]) if c["kind"] == "prompt" else 1
        total = int(old[b] + new[b])
        at = torch.arange(total - n, total, device=DEV)
        later = torch.arange(total, device=DEV)[None] > at[:, None]
        for h in range(Hkv):
            k, v = _token_rows(s, b, h, total, "k"), _token_rows(s, b, h, total, "v")
            for j in range(G):
                x = (q[row:row + n, h, j] @ k.T) * c["D"] ** -0.5
                x[later] = -math.inf
                l = torch.logsumexp(x, -1)
                out[row:row + n, h, j] = torch.exp(x - l[:, None]) @ v
                lse[row:row + n, h, j] = l
        row += n
    return out.view(-1, Hkv * G, D), lse.view(-1, Hkv * G)


def _exact_rope(s):
    c = s["case"]
    rot, page = c["rot"], c["page"]
    half = rot // 2
    first = [2 * i if c["pairs"] else i for i in range(half)]
    second = [2 * i + 1 if c["pairs"] else i + half for i in range(half)]
    angle = torch.stack([s["pos"][a].double() * float(w) for a, w in zip(s["axis"], s["inv"].tolist())], 1)
    z = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(x):
        x = x.double().clone()
        y = torch.complex(x[..., first], x[..., second]) * z
        x[..., first], x[..., second] = y.real, y.imag
        return x

    q, k = turned(s["q"]), turned(s["k"])
    if c["cache"] == "none":
        return q, k
    slots = s["slots"].long()
    outs, scales = [q], []
    for x in (k, s["v"].double()):
        pool = torch.zeros((s["P"], c["Hkv"], page, c["D"]), dtype=torch.float64, device=DEV)
        if c["cache"] == "fp8":
            top = x.abs().amax(-1)
            e = torch.where(top > 0, torch.ceil(torch.log2(top / 448)).clamp(-126, 127), 0)
            unit = torch.ones(pool.shape[:-1], dtype=torch.float64, device=DEV)
            unit[slots // page, :, slots % page] = torch.exp2(e)
            scales.append(unit)
            x = x / torch.exp2(e)[..., None]
        pool[slots // page, :, slots % page] = x
        outs.append(pool)
    return tuple(outs + scales)


def exact(case, seed):
    if case["kind"] == "pages":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(s)
    return _exact_attention(s, *lengths(case))
