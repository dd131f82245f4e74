"""Request-path operators on the GPU against their 64-bit restatements
(tests/request_oracle.py, which derives the bounds)."""
import math

import numpy as np
import pytest
import torch

from scope_amd import ops
from tests import request_oracle as R
from tests.gpu_pool import page_layout
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def same(got, want, what):
    got = got.cpu().numpy()
    assert np.array_equal(got, want), (what, np.argwhere(got != want)[:4].tolist())


# ---------------------------------------------------------------------------
# pages


def run_extend(table, lens, n_new, stack, free, page, P, N, base=None):
    t = ints(table)
    l, n, s, f = ints(lens), ints(n_new), ints(stack), ints([free])
    st = ops.pages_extend(t, l, n, s, f, page, P, N, pos_base=None if base is None else ints(base))
    want = R.extend(table, lens, n_new, stack, free, page, P, N, base)
    for got, w, what in zip((t, st.len_out, st.cu_new, st.positions, st.slots), want,
                            ("page_table", "len_out", "cu_new", "positions", "slots")):
        same(got, w, what)
    assert int(st.free_out) == want[5]
    same(l, np.asarray(lens), "len_in stays")
    same(f, np.asarray([free]), "free_in stays")
    return want


@pytest.mark.parametrize("B, page, top", [(1, 64, 1), (1, 64, 200), (3, 32, 70), (16, 64, 1), (64, 1, 9),
                                          (65, 48, 300), (257, 64, 5), (512, 128, 1000), (2048, 32, 40)])
def test_extend(B, page, top):
    rng = np.random.default_rng(B * 1000 + page)
    lens, n = rng.integers(0, 3 * top + 2, B), rng.integers(0, top + 1, B)
    table, used = page_layout(lens, page, B, spare=0)
    P = used + int(sum(-(-(l + k) // page) for l, k in zip(lens, n))) + 2
    table = np.concatenate([table, np.full((B, -(-top // page) + 1), -1, np.int32)], 1)
    stack = rng.permutation(np.arange(used, P)).astype(np.int32)
    run_extend(table, lens, n, stack, len(stack), page, P, int(n.sum()))
    # padding behind the last token, other positions than the partition's
    run_extend(table, lens, n, stack, len(stack), page, P, int(n.sum()) + 77, rng.integers(-9, 9999, B))


def test_extend_failures():
    """What does not fit gets nothing and takes nothing from those before it."""
    rng = np.random.default_rng(5)
    page, P, MP = 64, 30, 6
    table = rng.integers(0, P, (8, MP)).astype(np.int32)
    stack = rng.permutation(P).astype(np.int32)
    lens = [10, -1, 384, 383, 5, 64, 100, 0]
    n = [60, 3, 1, 1, -2, 0, 200, 129]
    N = sum(max(x, 0) for x in n)
    for free in (30, 7, 6, 5, 4, 1, 0, -3, 1000):  # (clamped to the stack)
        run_extend(table, lens, n, stack, free, page, P, N)
    run_extend(table, lens, n, stack, 30, page, P, N - 1)  # the last sequence's tokens do not fit the call
    run_extend(table, lens, n, stack, 30, page, P, 0)
    bad = stack.copy()
    bad[25:] = [-1, P, 1 << 30, 3, -7]
    run_extend(table, lens, n, bad, 30, page, P, N)  # page ids outside the pool: no slot
    table[0, 0] = P
    run_extend(table, lens, n, stack, 30, page, P, N)
    run_extend(np.zeros((0, 3), np.int32), [], [], stack, 30, page, P, 5)
    run_extend(table, [1 << 30] * 8, [1 << 30] * 8, stack, 30, page, P, 9)


@pytest.mark.parametrize("B, page", [(1, 64), (7, 32), (300, 64), (2048, 16)])
def test_release_and_reuse(B, page):
    rng = np.random.default_rng(B)
    lens = rng.integers(0, 500, B)
    table, used = page_layout(lens, page, B, spare=0)
    held = [-(-int(l) // page) for l in lens]
    done = rng.random(B) < 0.4
    done[-1] = True
    lens_in = lens.copy()
    if B > 5:
        lens_in[3], done[3], held[3] = -1, True, 0  # a failed sequence gives nothing back
    size = used + 3
    stack = np.full(size, -9, np.int32)
    s, f, t = ints(stack), ints([3]), ints(table)
    d = torch.from_numpy(done).to(DEV)
    len_out, free_out = ops.pages_release(t, ints(lens_in), d, s, f, page)
    back = [int(x) for b in range(B) if done[b] for x in table[b, :held[b]]]
    same(len_out, np.where(done, 0, lens_in), "len_out")
    same(s, np.array(([-9] * 3 + back + [-9] * size)[:size], np.int32), "stack")
    assert int(free_out) == 3 + len(back)
    same(t, table, "page_table stays")
    # a stack that is too small keeps what fits
    s2 = ints(stack[:5])
    _, f2 = ops.pages_release(t, ints(lens_in), d, s2, f, page)
    assert int(f2) == min(5, 3 + len(back))
    same(s2, np.array(([-9] * 3 + back + [-9] * 2)[:5], np.int32), "small stack")
    if B == 7:  # given back, handed out again from the top
        n = np.where(done, 70, 0)
        st = ops.pages_extend(t, len_out, ints(n), s, free_out, page, size, int(n.sum()))
        want = R.extend(table, len_out.cpu().numpy(), n, s.cpu().numpy(), int(free_out), page, size,
                        int(n.sum()))
        same(t, want[0], "table")
        same(st.slots, want[4], "slots")


# ---------------------------------------------------------------------------
# rotary


def rope_inputs(N, Hq, Hkv, D, rot, axes, seed, strided=True, far=1):
    g = torch.Generator().manual_seed(seed)
    qkv = bf16_randn((N, (Hq + 2 * Hkv) * D + 8 * strided), seed)
    q, k, v = (x.view(N, -1, D) if strided else x.contiguous().view(N, -1, D)
               for x in qkv[:, :(Hq + 2 * Hkv) * D].split((Hq * D, Hkv * D, Hkv * D), 1))
    pos = torch.randint(0, 40000 * far, (axes, N), generator=g, dtype=torch.int32)
    inv = (1e6 ** (-torch.arange(rot // 2) / (rot // 2))).float()
    axis = [int(a) for a in torch.randint(0, axes, (rot // 2,), generator=g)]
    return q, k, v, pos, inv, axis


def to_dev(*ts):
    """On the GPU with their strides (a slice of a fused tensor stays one)."""
    out = []
    for t in ts:
        d = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=DEV)
        out.append(d.copy_(t))
    return out


def rope_bound(x, rot, adjacent, factor):
    """fp32 work on the pair's two values: 2^-20 of their sizes (columns past rot
    are copied)."""
    a = x.double().abs() * abs(factor)
    t = torch.zeros_like(a)
    half = rot // 2
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if adjacent else (slice(0, half), slice(half, rot))
    t[..., one] = t[..., two] = (a[..., one] + a[..., two]) * 2.0 ** -20
    return t


@pytest.mark.parametrize("N, Hq, Hkv, D, rot, axes, adjacent, strided", [
    (1, 1, 1, 16, 16, 1, False, False), (3, 4, 2, 64, 64, 3, False, True), (5, 32, 8, 128, 128, 1, False, True),
    (7, 6, 2, 96, 64, 2, True, True), (2, 3, 1, 80, 80, 4, False, False), (9, 8, 8, 256, 256, 3, True, True),
    (33, 5, 5, 160, 48, 1, False, True), (2051, 2, 1, 64, 32, 3, False, True),
    (2048, 1, 1, 128, 128, 1, True, False), (4, 16, 4, 240, 240, 2, False, False)])
def test_rope(N, Hq, Hkv, D, rot, axes, adjacent, strided):
    q, k, _, pos, inv, axis = rope_inputs(N, Hq, Hkv, D, rot, axes, N + D, strided)
    dq, dk = to_dev(q, k)
    qo, ko = ops.rope(dq, dk, pos.to(DEV), inv.to(DEV), pair_axis=axis, adjacent=adjacent, factor=1.25)
    for x, got, what in ((q, qo, "q"), (k, ko, "k")):
        want = R.rotate(x, pos, inv, axis, adjacent, 1.25)
        R.check(got, want, want.abs() * 2.0 ** -8 + rope_bound(x, rot, adjacent, 1.25), what)
        assert torch.equal(got[..., rot:].cpu(), x[..., rot:])
    if not strided:  # in place
        ops.rope(dq, dk, pos.to(DEV), inv.to(DEV), pair_axis=axis, adjacent=adjacent, factor=1.25,
                 q_out=dq, k_out=dk)
        assert torch.equal(dq, qo) and torch.equal(dk, ko)


def test_rope_far_and_negative_positions():
    """Positions to 2^30: the angle is reduced in 64 bits (32 bits would be off by
    whole turns)."""
    q, k, _, pos, inv, _ = rope_inputs(40, 2, 1, 64, 64, 1, 3, far=26000)
    pos[0, :3] = torch.tensor([0, -1, -(1 << 30)], dtype=torch.int32)
    qo, ko = ops.rope(*to_dev(q, k), pos[0].contiguous().to(DEV), inv.to(DEV))
    for x, got in ((q, qo), (k, ko)):
        want = R.rotate(x, pos, inv, None, False)
        R.check(got, want, want.abs() * 2.0 ** -8 + rope_bound(x, 64, False, 1.0), "far")


def fresh_pools(P, Hkv, page, D, bits):
    """Pools full of a known pattern (the write must leave other slots alone)."""
    if bits == 16:
        return [torch.full((P, Hkv, page, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)] + \
            [None, None]
    byte = lambda v, *s: torch.full(s, v, dtype=torch.uint8, device=DEV)
    return [byte(0x31, P, Hkv, page, D).view(R.E4M3) for _ in range(2)] + \
        [byte(99, P, Hkv, page).view(R.E8M0) for _ in range(2)]


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("N, Hq, Hkv, D, rot, page, adjacent", [
    (1, 2, 1, 16, 16, 32, False), (5, 32, 8, 128, 128, 64, False), (37, 6, 2, 96, 64, 32, True),
    (70, 3, 3, 80, 80, 48, False), (9, 4, 4, 256, 128, 64, True), (2050, 2, 2, 64, 64, 64, False)])
def test_rope_append(bits, N, Hq, Hkv, D, rot, page, adjacent):
    q, k, v, pos, inv, axis = rope_inputs(N, Hq, Hkv, D, rot, 3, N * 3 + D)
    P = -(-N // page) + 3
    rng = np.random.default_rng(N)
    slots = rng.permutation(P * page)[:N].astype(np.int32)
    if N > 4:
        slots[[1, 3]] = [-1, P * page]  # no place
    pools = fresh_pools(P, Hkv, page, D, bits)
    before = [None if t is None else t.view(torch.uint8).cpu() for t in pools]
    qo = ops.rope_append(*to_dev(q, k, v), pos.to(DEV), inv.to(DEV), ints(slots), *pools,
                         pair_axis=axis, adjacent=adjacent)
    kr = R.rotate(k, pos, inv, axis, adjacent)
    want = R.rotate(q, pos, inv, axis, adjacent)
    R.check(qo, want, want.abs() * 2.0 ** -8 + rope_bound(q, rot, adjacent, 1.0), "q")
    put = (slots >= 0) & (slots < P * page)
    pid, off = torch.from_numpy(slots[put] // page).long(), torch.from_numpy(slots[put] % page).long()
    for i, (x, work) in enumerate(((kr[put], rope_bound(k, rot, adjacent, 1.0)[put]),
                                   (v.double()[put], torch.zeros_like(kr)[put]))):
        got = pools[i].cpu()
        if bits == 16:
            R.check(got[pid, :, off], x, x.abs() * 2.0 ** -8 + work, "kv"[i])
        else:
            s = pools[2 + i].cpu().view(torch.uint8)[pid, :, off].view(R.E8M0)
            val = R.dequantise(got.view(torch.uint8)[pid, :, off].view(R.E4M3), s)
            unit = s.double()[..., None]
            R.check(val, x, torch.maximum(x.abs() * 2.0 ** -4, unit * 2.0 ** -10) + work, "kv"[i])
            top = x.abs().amax(-1, keepdim=True)  # the least power of two that holds the row
            slack = 2.0 ** -20
            assert bool((top <= 448 * unit * (1 + slack)).all()), "scale too small"
            assert bool((top * (1 + slack) > 224 * unit).all()), "scale too large"
            if i == 1:  # values are not computed on: bit for bit
                wq, ws = R.quantise(v.double()[put])
                assert torch.equal(got.view(torch.uint8)[pid, :, off], wq.view(torch.uint8))
                assert torch.equal(s.view(torch.uint8), ws.view(torch.uint8))
    # everything else is as it was
    for t, b in zip(pools, before):
        if t is None:
            continue
        a = t.view(torch.uint8).cpu()
        b[pid, :, off] = a[pid, :, off]
        assert torch.equal(a, b), "slots that no token has changed"


def test_rope_append_odd_rows():
    """8-bit rows of zeros, of very small and large values, and with an infinity or a NaN."""
    D, Hkv = 64, 1
    v = bf16_randn((8, Hkv, D), 5)
    v[0] = 0
    v[1] *= 1e-38
    v[2] *= 1e37
    v[3, 0, 7] = float("inf")
    v[4, 0, 9] = float("nan")
    v[5] = 448.0
    v[6] = 450.0  # 448 is the largest that fits a scale of 1
    v[7, 0, 0] = 2.0 ** -133  # a denormal beside ones: flushed by the row's scale
    q = torch.zeros((8, 1, D), dtype=torch.bfloat16)
    pools = fresh_pools(1, Hkv, 32, D, 8)
    ops.rope_append(*to_dev(q, v, v), torch.zeros(8, dtype=torch.int32, device=DEV),
                    torch.ones(32, device=DEV), ints(np.arange(8)), *pools)
    wq, ws = R.quantise(v.double())
    for i in (0, 1):  # position 0: the keys do not turn either
        got, s = pools[i].view(torch.uint8).cpu()[0, 0, :8], pools[2 + i].view(torch.uint8).cpu()[0, 0, :8]
        fine = [0, 1, 2, 5, 6, 7]
        assert s[fine].tolist() == ws.view(torch.uint8)[fine, 0].tolist()
        # (0 and -0 of a flushed value are the same number)
        a, b = got.view(R.E4M3).float()[fine], wq.float()[fine, 0]
        assert torch.equal(a, b)
        assert s[[3, 4]].tolist() == [255, 255] and bool(got.view(R.E4M3).float()[[3, 4]].isnan().all())


# ---------------------------------------------------------------------------
# attention


def pools_of(lens, Hkv, D, page, bits, seed, sigma=1.0):
    """Pools whose slots that no token has are NaN, on the CPU and the GPU."""
    table, P = page_layout(lens, page, seed)
    slots = [int(table[b, t // page]) * page + t % page for b, L in enumerate(lens) for t in range(L)]
    cpu = []
    for i in range(2):
        x = bf16_randn((len(slots), Hkv, D), seed * 7 + i, sigma)
        pid, off = torch.tensor(slots).long() // page, torch.tensor(slots).long() % page
        if bits == 16:
            pool = torch.full((P, Hkv, page, D), math.nan, dtype=torch.bfloat16)
            pool[pid, :, off] = x
            cpu.append((pool, None))
        else:
            # rows of very different sizes
            g = torch.Generator().manual_seed(seed + i)
            x = x.float() * torch.exp2(torch.randint(-3, 3, (len(slots), Hkv, 1), generator=g).float())
            wq, ws = R.quantise(x)
            pool = torch.full((P, Hkv, page, D), 0x7f, dtype=torch.uint8)
            sc = torch.full((P, Hkv, page), 255, dtype=torch.uint8)
            pool[pid, :, off], sc[pid, :, off] = wq.view(torch.uint8), ws.view(torch.uint8)
            cpu.append((pool.view(R.E4M3), sc.view(R.E8M0)))
    (k, ks), (v, vs) = cpu
    dev = [t.to(DEV) if t is not None else None for t in (k, v, ks, vs)]
    return table, P, (k, v, ks, vs), dev


def decode_want(q, cpu, table, lens, page, Hkv, scale):
    B, Hq, D = q.shape
    G = Hq // Hkv
    res = [torch.zeros((B, Hq, D), dtype=torch.float64), torch.zeros((B, Hq), dtype=torch.float64),
           torch.zeros((B, Hq, D), dtype=torch.float64), torch.zeros((B, Hq), dtype=torch.float64)]
    k, v, ks, vs = cpu
    for b, L in enumerate(lens):
        for h in range(Hkv):
            kk, vv = (R.tokens_of(p, s, table[b], h, L, page) for p, s in ((k, ks), (v, vs)))
            for r, x in zip(res, R.attend(q[b, h * G:(h + 1) * G].double(), kk, vv, [L] * G, scale)):
                r[b, h * G:(h + 1) * G] = x
    return res


@pytest.mark.parametrize("D, Hkv, G, page, lens, splits", [
    (128, 2, 4, 64, [1], 0), (128, 2, 4, 64, [31, 32, 33, 0, 64, 65], 0), (64, 3, 5, 32, [200, 1, 7], 3),
    (32, 1, 16, 32, [99], 1), (96, 2, 3, 96, [300, 17], 7), (160, 1, 7, 64, [129, 500], 4),
    (192, 2, 1, 64, [70, 71, 72], 0), (224, 1, 2, 32, [33, 1], 1), (256, 2, 8, 64, [257, 5], 6),
    (128, 1, 8, 64, [3000], 64), (64, 2, 1, 64, [40] * 70, 0), (128, 1, 1, 32, [5] * 300, 0),
    (128, 4, 2, 128, [1500, 0, 3, 900], 17)])
def test_decode8(D, Hkv, G, page, lens, splits):
    table, P, cpu, dev = pools_of(lens, Hkv, D, page, 8, D + len(lens))
    B, Hq = len(lens), Hkv * G
    q, scale = bf16_randn((B, Hq, D), 9), D ** -0.5
    want_o, want_l, tol_o, tol_l = decode_want(q, cpu, table, lens, page, Hkv, scale)
    args = (q.to(DEV), *dev, ints(table), ints(lens), scale, max(lens), splits)
    out, lse = ops.gqa8_decode_partial(*args)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    o16, l16 = ops.gqa8_decode_full(*args)
    R.check(o16, want_o, tol_o + want_o.abs() * 2.0 ** -8, "bf16 out")
    R.check(l16, want_l, tol_l, "lse")
    again, _ = ops.gqa8_decode_partial(*args)
    assert torch.equal(again, out)


def test_decode8_scale_extremes_and_bad_scales():
    """Scales over e8m0's range (the products stay in bf16's), and a NaN scale."""
    D, page, L = 64, 32, 40
    table, P, cpu, _ = pools_of([L], 1, D, page, 8, 3)
    k, v, ks, vs = (t.clone() for t in cpu)
    rows = [(int(table[0, t // page]), t % page) for t in range(L)]
    vb, kb = vs.view(torch.uint8), ks.view(torch.uint8)
    for i, (p, o) in enumerate(rows):
        vb[p, 0, o] = [1, 60, 127, 200, 230][i % 5]
        kb[p, 0, o] = [0, 1, 100, 127, 128][i % 5]
    q = bf16_randn((1, 2, D), 4)

    def run():
        dev = [t.to(DEV) for t in (k, v, ks, vs)]
        return ops.gqa8_decode_partial(q.to(DEV), *dev, ints(table), ints([L]), 0.1, L)

    want_o, want_l, tol_o, tol_l = decode_want(q, (k, v, ks, vs), table, [L], page, 1, 0.1)
    out, lse = run()
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    for t in (kb, vb):
        p, o = rows[33]
        keep = int(t[p, 0, o])
        t[p, 0, o] = 255
        assert bool(run()[0].isnan().all())
        t[p, 0, o] = keep


def test_decode8_bad_pages_and_lengths():
    lens = [100, 70, 40, 0, 64]
    table, P, cpu, dev = pools_of(lens, 2, 64, 32, 8, 21)
    q = bf16_randn((5, 4, 64), 2)
    want = decode_want(q, cpu, table, lens, 32, 2, 0.125)
    table[0, 3] = P        # reached
    table[1, 0] = -5       # reached
    table[2, 2:] = 1 << 30  # not reached by 40 tokens
    lens[4] = 32 * table.shape[1] + 1  # past the row's capacity
    for fn in (ops.gqa8_decode_partial, ops.gqa8_decode_full):
        for splits in (1, 5, 0):
            out, lse = fn(q.to(DEV), *dev, ints(table), ints(lens), 0.125, 100, splits)
            assert bool(out[[0, 1, 4]].isnan().all()) and bool(lse[[0, 1, 4]].isnan().all())
            half = 2.0 ** -8 if out.dtype == torch.bfloat16 else 0.0
            R.check(out[2:4], want[0][2:4], want[2][2:4] + want[0][2:4].abs() * half, "fine ones")
            R.check(lse[2:4], want[1][2:4], want[3][2:4], "fine ones")
    out, lse = ops.gqa8_decode_partial(q.to(DEV), *dev, ints(table), ints([-1] * 5), 0.125, 100)
    assert bool(out.isnan().all()) and bool(lse.isnan().all())


def prompt_want(q, cpu, table, lens, new, page, Hkv, scale, c0=0):
    N, Hq, D = q.shape
    G = Hq // Hkv
    res = [torch.zeros((N, Hq, D), dtype=torch.float64), torch.zeros((N, Hq), dtype=torch.float64),
           torch.zeros((N, Hq, D), dtype=torch.float64), torch.zeros((N, Hq), dtype=torch.float64)]
    k, v, ks, vs = cpu
    at = c0
    for b, (L, n) in enumerate(zip(lens, new)):
        vis = [max(0, L - n + i + 1) for i in range(n)]
        for h in range(Hkv):
            kk, vv = (R.tokens_of(p, s, table[b], h, L, page) for p, s in ((k, ks), (v, vs)))
            for g in range(G):
                for r, x in zip(res, R.attend(q[at:at + n, h * G + g].double(), kk, vv, vis, scale)):
                    r[at:at + n, h * G + g] = x
        at += n
    return res


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("D, Hkv, G, page, lens, new, splits", [
    (128, 1, 1, 32, [1], [1], 0), (128, 2, 4, 64, [65, 64, 1, 33], [65, 3, 1, 32], 0),
    (64, 2, 3, 32, [300, 17, 128], [130, 0, 128], 0), (96, 1, 5, 96, [200, 0, 90], [77, 0, 1], 0),
    (32, 1, 2, 32, [150], [150], 0), (160, 1, 1, 64, [140], [133], 0), (192, 1, 2, 64, [100, 30], [100, 7], 0),
    (224, 1, 1, 32, [97], [33], 0), (256, 1, 2, 64, [150, 3], [70, 3], 0),
    (128, 2, 4, 64, [700], [5], 0), (128, 1, 4, 64, [900, 400], [3, 2], 7), (64, 1, 40, 64, [70, 200], [2, 9], 0),
    (128, 1, 2, 128, [500], [200], 3), (64, 1, 1, 32, [3] * 150, [2] * 150, 0),
    (128, 2, 1, 64, [10, 5], [30, 5], 0), (96, 1, 2, 32, [400], [5], 64), (256, 1, 1, 32, [300], [4], 5)])
def test_prompt(bits, D, Hkv, G, page, lens, new, splits):
    """(30 queries of a 10-token partition: the first 20 see nothing.)"""
    table, P, cpu, dev = pools_of(lens, Hkv, D, page, bits, D + len(lens))
    k, v, ks, vs = dev
    N, Hq = sum(new), Hkv * G
    q, scale = bf16_randn((N, Hq, D), 9), D ** -0.5
    want_o, want_l, tol_o, tol_l = prompt_want(q, cpu, table, lens, new, page, Hkv, scale)
    args = (q.to(DEV), k, v, ints(table), ints(lens), ints(np.concatenate([[0], np.cumsum(new)])), scale,
            max(lens))
    kw = dict(k_scale=ks, v_scale=vs, n_splits=splits)
    out, lse = ops.gqa_prompt(*args, out_dtype=torch.float32, **kw)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    o16, none = ops.gqa_prompt(*args, want_lse=False, **kw)
    assert none is None
    R.check(o16, want_o, tol_o + want_o.abs() * 2.0 ** -8, "bf16 out")


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("splits", (0, 1, 4))
@pytest.mark.parametrize("D, G, lens, new", [
    # rows of more than one wave and up to two, on average
    (32, 3, [700, 90], [14, 9]), (64, 7, [64, 900, 31], [9, 6, 4]), (96, 2, [520, 33], [32, 20]),
    (128, 4, [1000, 40, 65], [16, 9, 11]), (160, 3, [300, 310], [20, 12]), (256, 8, [290, 64], [7, 5]),
    # few on average, but many of one sequence
    (128, 1, [400, 9, 5, 70, 33, 32, 64], [300, 1, 0, 3, 2, 1, 1]), (64, 2, [200] + [40] * 12, [150] + [1] * 12)])
def test_prompt_few_rows(bits, splits, D, G, lens, new):
    page = 64
    table, P, cpu, (k, v, ks, vs) = pools_of(lens, 2, D, page, bits, 31 + D)
    q, scale = bf16_randn((sum(new), 2 * G, D), 8), D ** -0.5
    want_o, want_l, tol_o, tol_l = prompt_want(q, cpu, table, lens, new, page, 2, scale)
    out, lse = ops.gqa_prompt(q.to(DEV), k, v, ints(table), ints(lens),
                              ints(np.concatenate([[0], np.cumsum(new)])), scale, max(lens), ks, vs,
                              n_splits=splits, out_dtype=torch.float32)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


def test_prompt_packed_elsewhere():
    """Rows before the first and behind the last sequence keep what they held, at any
    split count."""
    lens, new, page, D = [70, 40], [9, 40], 32, 64
    table, P, cpu, (k, v, _, _) = pools_of(lens, 1, D, page, 16, 5)
    q = bf16_randn((60, 2, D), 1)
    want_o, want_l, tol_o, tol_l = prompt_want(q, cpu, table, lens, new, page, 1, 0.1, c0=4)
    for splits in (1, 2):
        out, lse = torch.full((60, 2, D), 5.0, device=DEV), torch.full((60, 2), 6.0, device=DEV)
        ops.gqa_prompt(q.to(DEV), k, v, ints(table), ints(lens), ints([4, 13, 53]), 0.1, 70, out=out,
                       lse=lse, n_splits=splits)
        R.check(out[4:53], want_o[4:53], tol_o[4:53], "out")
        R.check(lse[4:53], want_l[4:53], tol_l[4:53], "lse")
        for x, was in ((out, 5.0), (lse, 6.0)):
            assert bool((x[:4] == was).all()) and bool((x[53:] == was).all())


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("n, G, splits", [(60, 2, 0), (150, 2, 1), (3, 2, 2)])
@pytest.mark.parametrize("where", ("k", "v"))
def test_prompt_nonfinite_tokens(bits, n, G, splits, where):
    """An infinity or a NaN in a token's key or value reaches the rows that see it and
    no other."""
    L, page, D = 200, 64, 64
    table, P, cpu, _ = pools_of([L], 1, D, page, bits, 31)
    k, v, ks, vs = (t.clone() if t is not None else None for t in cpu)
    at = L - n // 2 - 1
    pool = k if where == "k" else v
    pid, off = int(table[0, at // page]), at % page
    if bits == 16:
        pool[pid, 0, off, 5] = math.inf if n == 60 else math.nan
    else:
        pool.view(torch.uint8)[pid, 0, off, 5] = 0x7f
    q = bf16_randn((n, G, D), 3)
    dev = [t.to(DEV) if t is not None else None for t in (k, v, ks, vs)]
    out, lse = ops.gqa_prompt(q.to(DEV), dev[0], dev[1], ints(table), ints([L]), ints([0, n]), 0.125, L,
                              k_scale=dev[2], v_scale=dev[3], n_splits=splits, out_dtype=torch.float32)
    want_o, want_l, tol_o, tol_l = prompt_want(q, (k, v, ks, vs), table, [L], [n], page, 1, 0.125)
    clean = at - (L - n)  # rows before it
    assert clean > 0
    R.check(out[:clean], want_o[:clean], tol_o[:clean], "rows that do not see it")
    R.check(lse[:clean], want_l[:clean], tol_l[:clean], "rows that do not see it")
    got, want = out[clean:].cpu(), want_o[clean:]
    if where == "v":
        assert torch.equal(got.isfinite()[..., 5], torch.zeros_like(got[..., 5], dtype=torch.bool))
        cols = [c for c in range(D) if c != 5]
        R.check(got[..., cols], want[..., cols], tol_o[clean:][..., cols], "other columns")
        R.check(lse[clean:], want_l[clean:], tol_l[clean:], "lse")
    elif bits == 8 or n != 60:
        assert bool(got.isnan().all()) and bool(lse[clean:].isnan().all())


def test_prompt_scale_signs():
    """A negative scale, and zero (the mean of what a row sees)."""
    lens, new, page, D = [90], [40], 32, 64
    table, P, cpu, (k, v, _, _) = pools_of(lens, 1, D, page, 16, 8)
    q = bf16_randn((40, 2, D), 1)
    for scale in (-0.2, 0.0):
        for splits in (1, 2):
            want_o, want_l, tol_o, tol_l = prompt_want(q, cpu, table, lens, new, page, 1, scale)
            out, lse = ops.gqa_prompt(q.to(DEV), k, v, ints(table), ints(lens), ints([0, 40]), scale, 90,
                                      n_splits=splits, out_dtype=torch.float32)
            R.check(out, want_o, tol_o, f"out at scale {scale}")
            R.check(lse, want_l, tol_l, f"lse at scale {scale}")


def test_prompt_large_scores():
    """Scores of hundreds: the running maximum moves, weights underflow."""
    lens, new, page, D = [300], [100], 32, 64
    table, P, cpu, (k, v, _, _) = pools_of(lens, 1, D, page, 16, 12, sigma=6.0)
    q = bf16_randn((100, 1, D), 1, 4.0)
    want_o, want_l, tol_o, tol_l = prompt_want(q, cpu, table, lens, new, page, 1, 1.0)
    out, lse = ops.gqa_prompt(q.to(DEV), k, v, ints(table), ints(lens), ints([0, 100]), 1.0, 300,
                              out_dtype=torch.float32)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


@pytest.mark.parametrize("splits", (1, 3))
def test_prompt_bad_pages_and_lengths(splits):
    lens, new, page, D = [150, 100, 64, 80, 10], [100, 5, 64, 4, 3], 32, 64
    table, P, cpu, (k, v, _, _) = pools_of(lens, 2, D, page, 16, 77)
    N = sum(new)
    q = bf16_randn((N, 4, D), 2)
    want_o, want_l, tol_o, tol_l = prompt_want(q, cpu, table, lens, new, page, 2, 0.125)
    table[0, 3] = P   # tokens 96 .. 127: seen by queries from position 96 on
    table[1, 0] = -1  # seen by every query
    table[2, 2:] = 1 << 30  # never reached
    lens[3], lens[4] = -1, page * table.shape[1] + 1
    cu = np.concatenate([[0], np.cumsum(new)])
    out, lse = ops.gqa_prompt(q.to(DEV), k, v, ints(table), ints(lens), ints(cu), 0.125, 150,
                              n_splits=splits, out_dtype=torch.float32)
    first = 96 - 50  # the query at position 96
    fine = list(range(first)) + list(range(cu[2], cu[3]))
    R.check(out[fine], want_o[fine], tol_o[fine], "fine rows")
    R.check(lse[fine], want_l[fine], tol_l[fine], "fine rows")
    gone = [i for i in range(N) if i not in fine]
    assert bool(out[gone].isnan().all()) and bool(lse[gone].isnan().all())


def test_refused_tensors():
    t = torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    l = torch.zeros(2, dtype=torch.int32, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device=DEV)
    pos, inv = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(32, device=DEV)
    pool = torch.zeros((3, 2, 32, 64), dtype=torch.bfloat16, device=DEV)
    p8, s8 = fresh_pools(3, 2, 32, 64, 8)[::2]
    with pytest.raises(TypeError, match="len_in"):
        ops.pages_extend(t, l.long(), l, l, one, 32, 3, 4)
    with pytest.raises(ValueError, match="B"):
        ops.pages_extend(t, one, l, l, one, 32, 3, 4)
    with pytest.raises(TypeError, match="done"):
        ops.pages_release(t, l, l, l, one, 32)
    with pytest.raises(ValueError, match="contiguous"):
        ops.rope(x.transpose(0, 1).contiguous().transpose(0, 1), x, pos, inv)
    with pytest.raises(ValueError, match="positions"):
        ops.rope(x, x, pos[:3], inv)
    with pytest.raises(ValueError, match="pair_axis"):
        ops.rope(x, x, pos, inv, pair_axis=[0] * 31)
    with pytest.raises(ops.WsError, match="axis"):
        ops.rope(x, x, pos, inv, pair_axis=[1] * 32)
    with pytest.raises(ValueError, match="both"):
        ops.rope_append(x, x, x, pos, inv, pos, p8.view(torch.bfloat16), p8.view(torch.bfloat16), v_scale=s8)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.rope_append(x, x, x, pos, inv, pos, pool, pool, s8, s8)
    with pytest.raises(ValueError, match="do not match"):
        ops.rope_append(x, x[:, :1], x, pos, inv, pos, pool, pool)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.gqa8_decode_partial(x[:2], pool, pool, s8, s8, t, l, 1.0, 3)
    with pytest.raises(ValueError, match="both"):
        ops.gqa8_decode_partial(x[:2], p8, p8, None, None, t, l, 1.0, 3)
    with pytest.raises(ValueError, match="match"):
        ops.gqa_prompt(x.view(4, 4, 32), pool, pool, t, l, pos[:3], 1.0, 3)
    with pytest.raises(ValueError, match="cu_new"):
        ops.gqa_prompt(x, pool, pool, t, l, l, 1.0, 3)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        ops.gqa_prompt(x, pool, pool, t, l, pos[:3], 1.0, 3, out_dtype=torch.float16)


@pytest.mark.parametrize("bits", (16, 8))
def test_pools_past_4_gib(bits):
    """The same pages at the far end of pools of more than 2^32 bytes: the same bits."""
    D, Hkv, page, lens, new = 256, 2, 64, [200, 90], [40, 3]
    table, P, _, small = pools_of(lens, Hkv, D, page, bits, 77)
    Pb = 70000 * 16 // bits
    shift = Pb - P
    far = np.where(table >= 0, table + shift, table).astype(np.int32)
    big = [None if t is None else torch.zeros((Pb,) + t.shape[1:], dtype=torch.uint8, device=DEV).view(t.dtype)
           if t.element_size() == 1 else torch.zeros((Pb,) + t.shape[1:], dtype=t.dtype, device=DEV)
           for t in small]
    assert big[0].numel() * big[0].element_size() > 1 << 32

    def raw(t):
        return t.view(torch.uint8)

    N = 50
    q, k, v = (bf16_randn((N, h, D), 5 + i).to(DEV) for i, h in enumerate((4, Hkv, Hkv)))
    pos, inv = ints(np.arange(N)), (1e4 ** (-torch.arange(D // 2) / (D // 2))).float().to(DEV)
    slots = np.array([int(table[0, t // page]) * page + t % page for t in range(100, 100 + N)])
    for pools, t, s in ((small, table, slots), (big, far, slots + shift * page)):
        if pools is big:
            for a, b in zip(pools, start):
                if a is not None:
                    raw(a)[shift:] = raw(b)
        else:
            start = [None if x is None else x.clone() for x in small]
        ops.rope_append(q, k, v, pos, inv, ints(s), *pools)
    for a, b in zip(big, small):
        if a is not None:
            assert torch.equal(raw(a)[shift:], raw(b)) and not bool(a.view(torch.int32)[:shift].any())
    q = q[:sum(new)]
    calls = [lambda p, t: ops.gqa_prompt(q, p[0], p[1], ints(t), ints(lens), ints([0, 40, 43]), 0.1, 200, p[2], p[3])]
    if bits == 8:
        calls.append(lambda p, t: ops.gqa8_decode_partial(q[:2], *p, ints(t), ints(lens), 0.1, 200))
    for call in calls:
        for x, y in zip(call(small, table), call(big, far)):
            assert bool(x.isfinite().all()) and torch.equal(x, y)


@pytest.mark.parametrize("bits", (8, 16))
@pytest.mark.parametrize("B, Hkv", [(256, 2), (256, 1), (300, 1)])
def test_decode_at_a_long_capacity(bits, B, Hkv):
    """Many sequences, one of them long, with the row's capacity as max_len (a captured
    step's): the worst case is millions of blocks, the lengths are a few hundred."""
    D, G, page, cap = 64, 2, 64, 1 << 17
    lens = [int(x) for x in np.random.default_rng(B).integers(0, 70, B)]
    lens[B // 3] = 4100
    table, P, cpu, (k, v, ks, vs) = pools_of(lens, Hkv, D, page, bits, B + Hkv)
    table = np.concatenate([table, np.full((B, cap // page - table.shape[1]), -1, np.int32)], 1)
    q = bf16_randn((B, G * Hkv, D), 4)
    want_o, want_l, tol_o, tol_l = decode_want(q, cpu, table, lens, page, Hkv, 0.125)
    if bits == 8:
        out, lse = ops.gqa8_decode_partial(q.to(DEV), k, v, ks, vs, ints(table), ints(lens), 0.125, cap)
    else:
        out, lse = ops.gqa_decode_partial(q.to(DEV), k, v, ints(table), ints(lens), 0.125, cap)
        tol_o = 2 * tol_o  # bf16 pieces: each off by another 2^-8 of its own weighted sum of |v|
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


def prompt_on(q, dev, table, lens, new, scale, **kw):
    return ops.gqa_prompt(q.to(DEV), dev[0], dev[1], ints(table), ints(lens),
                          ints(np.concatenate([[0], np.cumsum(new)])), scale, max(lens), dev[2], dev[3],
                          out_dtype=torch.float32, **kw)


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("L, n, D", [(2090, 3, 64), (2130, 70, 64), (2165, 5, 96), (4230, 2, 64), (4200, 130, 64),
                                     (2300, 9, 256)])
def test_prompt_windows_of_page_ids(bits, L, n, D):
    """One workgroup walks more than 64 tiles: its window of page ids is fetched again, with
    0 to 3 steps behind the last whole turn; a bad page in a later window is seen."""
    page, G = 32, 2
    table, P, cpu, dev = pools_of([L, 50], 1, D, page, bits, L + n)
    new = [n, 1]
    q, scale = bf16_randn((n + 1, G, D), 2), D ** -0.5
    want_o, want_l, tol_o, tol_l = prompt_want(q, cpu, table, [L, 50], new, page, 1, scale)
    out, lse = prompt_on(q, dev, table, [L, 50], new, scale, n_splits=1)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    table[0, 65] = P + 3  # (a page a tile; seen by every row)
    out, lse = prompt_on(q, dev, table, [L, 50], new, scale, n_splits=1)
    if L - n >= 66 * 32:
        assert bool(out[:n].isnan().all()) and bool(lse[:n].isnan().all())
    else:  # the rows that see its first token
        seen = 65 * 32 - (L - n)
        R.check(out[:max(seen, 0)], want_o[:max(seen, 0)], tol_o[:max(seen, 0)], "rows before the bad page")
        assert bool(out[max(seen, 0):n].isnan().all()) and bool(lse[max(seen, 0):n].isnan().all())
    R.check(out[n:], want_o[n:], tol_o[n:], "the other sequence")


@pytest.mark.parametrize("D, Hkv, lens, splits", [
    (64, 1, [4500], 1), (128, 2, [2016, 2100, 40], 1), (96, 1, [2048, 1, 2080, 4129], 2), (256, 1, [2044, 33, 4500], 1),
    (64, 3, [2080, 31, 0, 4100], 3)])
def test_decode8_windows_of_page_ids(D, Hkv, lens, splits):
    """A split of more than 64 blocks fetches its blocks' metadata again, with rows that end
    before, at and behind a window's edge; a bad page in a later window is seen."""
    page, G = 32, 2
    table, P, cpu, dev = pools_of(lens, Hkv, D, page, 8, sum(lens))
    q, scale = bf16_randn((len(lens), G * Hkv, D), 6), D ** -0.5
    want_o, want_l, tol_o, tol_l = decode_want(q, cpu, table, lens, page, Hkv, scale)
    args = lambda: (q.to(DEV), *dev, ints(table), ints(lens), scale, max(lens), splits)
    out, lse = ops.gqa8_decode_partial(*args())
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    b = int(np.argmax(lens))
    table[b, -(-lens[b] // page) - 1] = P  # its last page
    out, lse = ops.gqa8_decode_partial(*args())
    assert bool(out[b].isnan().all()) and bool(lse[b].isnan().all())
    for i in range(len(lens)):
        if i != b:
            R.check(out[i], want_o[i], tol_o[i], "the other sequences")


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("B, splits", [(70, 3), (70, 0), (300, 3), (300, 0), (129, 0)])
def test_prompt_many_split_sequences(bits, B, splits):
    """More sequences than a wave's lanes, split: both kernels number the pieces of a lane's
    sequences alike.  A few are long, so that they are split where the lengths decide."""
    D, page, G, rng = 32, 64, 2, np.random.default_rng(B)
    lens = rng.integers(1, 60, B)
    lens[rng.permutation(B)[:4]] = (700, 1500, 333, 900)
    new = np.minimum(lens, rng.integers(0, 5, B))
    new[int(np.argmax(lens))] = 40  # (bf16: three tiles of rows)
    table, P, cpu, dev = pools_of(lens, 1, D, page, bits, B)
    q = bf16_randn((int(new.sum()), G, D), 3)
    want_o, want_l, tol_o, tol_l = prompt_want(q, cpu, table, lens, new, page, 1, 0.2)
    out, lse = prompt_on(q, dev, table, lens, new, 0.2, n_splits=splits)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


@pytest.mark.parametrize("D, Hkv, G, lens, splits", [
    (128, 2, 4, [1], 0), (128, 2, 4, [31, 0, 33, 700], 0), (80, 1, 3, [200, 65], 3), (256, 2, 16, [257, 5], 6),
    (64, 2, 1, [40] * 70, 0), (16, 1, 2, [129], 1)])
def test_decode_full(D, Hkv, G, lens, splits):
    table, P, cpu, (k, v, _, _) = pools_of(lens, Hkv, D, 64, 16, D + len(lens))
    q, scale = bf16_randn((len(lens), Hkv * G, D), 9), D ** -0.5
    want_o, want_l, tol_o, tol_l = decode_want(q, cpu, table, lens, 64, Hkv, scale)
    args = (q.to(DEV), k, v, ints(table), ints(lens), scale, max(lens), splits)
    out, lse = ops.gqa_decode_full(*args)
    # bf16 pieces: each off by another 2^-8 of its own weighted sum of |v|; then the output's rounding
    R.check(out, want_o, 2 * tol_o + want_o.abs() * 2.0 ** -8, "out")
    R.check(lse, want_l, tol_l, "lse")
    part, part_l = ops.gqa_decode_partial(*args)
    assert torch.equal(out, part.bfloat16()) and torch.equal(lse, part_l)
    mine = torch.empty_like(out), torch.empty_like(lse)
    assert ops.gqa_decode_full(*args, *mine)[0] is mine[0] and torch.equal(mine[0], out)
    for bad, err, says in ((dict(out_bf16=part), TypeError, "out_bf16"), (dict(lse=lse[:, :1]), ValueError, "lse")):
        with pytest.raises(err, match=says):
            ops.gqa_decode_full(*args, **{**bad, **({"lse": bad["lse"].contiguous()} if "lse" in bad else {})})
    with pytest.raises(ValueError, match="match the pools"):
        ops.gqa_decode_full(q[..., :8].contiguous().to(DEV), *args[1:])
