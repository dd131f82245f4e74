"""The latent path's operators on the GPU against their 64-bit restatements
(tests/latent_oracle.py and tests/request_oracle.py, which derive the bounds)."""
import math

import numpy as np
import pytest
import torch

from scope_amd import ops
from tests import latent_oracle as L
from tests import request_oracle as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
C, PE, W = L.C, L.PE, L.W


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def dev(cpu):
    return [None if t is None else t.to(DEV) for t in cpu]


# ---------------------------------------------------------------------------
# the write


def inputs(N, H, seed, strided=True, sigma=1.0):
    """(c, pe, q_pe, positions, inv_freq): parts of a projection's rows, or tensors of their own."""
    kv, q = bf16_randn((N, W + 8 * strided), seed, sigma), bf16_randn((N, H, 192 if strided else PE), seed + 1)
    g = torch.Generator().manual_seed(seed)
    pos = torch.randint(0, 40000, (N,), generator=g, dtype=torch.int32)
    inv = (1e4 ** (-torch.arange(PE // 2) / (PE // 2))).float()
    c, pe, q = kv[:, :C], kv[:, C:W], q[..., 128:] if strided else q
    return (c, pe, q, pos, inv) if strided else (c.contiguous(), pe.contiguous(), q, pos, inv)


def on_gpu(*ts):
    """On the GPU with their strides (a part of a tensor stays one)."""
    out = []
    for t in ts:
        whole = torch.zeros(t.untyped_storage().size() // t.element_size(), dtype=t.dtype, device=DEV)
        d = whole.as_strided(t.shape, t.stride(), t.storage_offset())
        out.append(d.copy_(t))
    return out


def fresh(P, page, bits, block=1):
    """A pool full of a known pattern (the write must leave other slots alone)."""
    if bits == 16:
        return torch.full((P, page, W), 7.0, dtype=torch.bfloat16, device=DEV), None
    return (torch.full((P, page, W), 0x31, dtype=torch.uint8, device=DEV).view(R.E4M3),
            torch.full((P, page // block), 99, dtype=torch.uint8, device=DEV).view(R.E8M0))


def check_q(q, q_pe, pos, inv, adjacent, factor):
    want = R.rotate(q_pe, pos, inv, None, adjacent, factor)
    a = q_pe.double().abs() * abs(factor)
    one, two = (slice(0, PE, 2), slice(1, PE, 2)) if adjacent else (slice(0, PE // 2), slice(PE // 2, PE))
    work = torch.zeros_like(a)
    work[..., one] = work[..., two] = (a[..., one] + a[..., two]) * 2.0 ** -20
    R.check(q, want, want.abs() * 2.0 ** -8 + work, "q")


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("N, H, page, adjacent, norm, strided", [
    (1, 1, 32, False, None, False), (5, 16, 64, True, "bf16", True), (37, 20, 48, False, "f32", True),
    (2051, 3, 64, True, "bf16", True), (70, 128, 32, False, None, True)])
def test_append(bits, N, H, page, adjacent, norm, strided):
    c, pe, q_pe, pos, inv = inputs(N, H, N * 3 + H, strided)
    weight = None if norm is None else 1 + 0.2 * bf16_randn((C,), 9).float()
    if norm == "bf16":
        weight = weight.to(torch.bfloat16)
    P = -(-N // page) + 3
    slots = np.random.default_rng(N).permutation(P * page)[:N].astype(np.int32)
    if N > 4:
        slots[[1, 3]] = [-1, P * page]  # no place
    pool, scale = fresh(P, page, bits)
    before = pool.view(torch.uint8).cpu(), None if scale is None else scale.view(torch.uint8).cpu()
    args = on_gpu(c, pe, q_pe)
    q = ops.latent_rope_append(*args, pos.to(DEV), inv.to(DEV), ints(slots), pool, scale,
                               None if weight is None else weight.to(DEV), 1e-5, adjacent, 1.25)
    check_q(q, q_pe, pos, inv, adjacent, 1.25)
    x, work = L.latents(c, pe, pos, inv, adjacent, 1.25, weight, 1e-5)
    put = (slots >= 0) & (slots < P * page)
    pid, off = torch.from_numpy(slots[put] // page).long(), torch.from_numpy(slots[put] % page).long()
    x, work = x[put], work[put]
    got = pool.cpu()
    if bits == 16:
        R.check(got[pid, off], x, x.abs() * 2.0 ** -8 + work, "latent")
    else:
        s = scale.cpu().view(torch.uint8)[pid, off].view(R.E8M0)
        val, unit = R.dequantise(got.view(torch.uint8)[pid, off].view(R.E4M3), s), s.double()[:, None]
        R.check(val, x, torch.maximum(x.abs() * 2.0 ** -4, unit * 2.0 ** -10) + work, "latent")
        top = x.abs().amax(-1, keepdim=True)  # the least power of two that holds the row
        assert bool((top <= 448 * unit * (1 + 2.0 ** -16)).all()), "scale too small"
        assert bool((top * (1 + 2.0 ** -16) > 224 * unit).all()), "scale too large"
        if norm is None:  # c is not computed on: bit for bit
            codes = (x / unit).float().to(R.E4M3).view(torch.uint8)[:, :C]
            assert torch.equal(got.view(torch.uint8)[pid, off][:, :C], codes)
    for t, b in ((pool, before[0]), (scale, before[1])):
        if t is not None:  # everything else is as it was
            a = t.view(torch.uint8).cpu()
            b[pid, off] = a[pid, off]
            assert torch.equal(a, b), "slots that no token has changed"
    if not strided:  # in place
        ops.latent_rope_append(*args, pos.to(DEV), inv.to(DEV), ints(slots), pool, scale,
                               None if weight is None else weight.to(DEV), 1e-5, adjacent, 1.25, q_out=args[2])
        assert torch.equal(args[2], q)


@pytest.mark.parametrize("block, page, calls", [
    (32, 64, [[40, 0, 7], [1, 33, 60], [1, 1, 1], [25, 2, 0], [1, 1, 1]]),
    (64, 64, [[100, 1], [3, 1], [1, 70], [1, 1]]), (16, 48, [[5, 17, 0, 90], [1] * 4, [13, 0, 1, 200]]),
    (128, 128, [[300], [1], [100]]), (2, 32, [[7, 4], [1, 1], [1, 1], [3, 3]])])
def test_append_blocks(block, page, calls):
    """Several tokens to a scale, over calls that begin and end inside blocks: a scale is the
    least that holds its block's tokens and never falls while the block grows; where it
    rises, the older tokens are rounded again, and nothing else of them changes."""
    B, top = len(calls[0]), max(sum(c[b] for c in calls) for b in range(len(calls[0])))
    cols = -(-top // page)
    table = np.random.default_rng(page).permutation(B * cols + 2)[:B * cols].reshape(B, cols)
    pool, scale = fresh(B * cols + 2, page, 8, block)
    lens, rose = np.zeros(B, np.int64), 0
    for i, n_new in enumerate(calls):
        N = sum(n_new)
        c, pe, q_pe, pos, inv = inputs(N, 4, 50 + i, sigma=1.0 + 3 * i)  # later tokens are larger
        seq = np.repeat(np.arange(B), n_new)
        tok = np.concatenate([np.arange(lens[b], lens[b] + n) for b, n in enumerate(n_new)])
        slots = table[seq, tok // page] * page + tok % page
        was, was_s = pool.view(torch.uint8).cpu().view(-1, W), scale.view(torch.uint8).cpu().view(-1)
        q = ops.latent_rope_append(*on_gpu(c, pe, q_pe), pos.to(DEV), inv.to(DEV), ints(slots), pool, scale)
        check_q(q, q_pe, pos, inv, False, 1.0)
        x, work = L.latents(c, pe, pos, inv, False, 1.0, None, 0.0)
        got, got_s = pool.view(torch.uint8).cpu().view(-1, W), scale.view(torch.uint8).cpu().view(-1)
        codes, scales = was.clone(), was_s.clone()
        blocks = slots // block
        for k in np.unique(blocks):
            mine = blocks == k
            first = int(slots[mine].min() - k * block)
            big = float(x[mine].abs().max())
            byte = int(got_s[k])
            low = int(was_s[k]) if first > 0 else 0
            assert byte >= low and big <= 448 * 2.0 ** (byte - 127) * (1 + 2.0 ** -16)
            assert byte == low or big * (1 + 2.0 ** -16) > 224 * 2.0 ** (byte - 127), "scale too large"
            scales[k] = byte
            unit = 2.0 ** (byte - 127)
            val = got[slots[mine]].view(R.E4M3).double() * unit
            R.check(val, x[mine], torch.maximum(x[mine].abs() * 2.0 ** -4, torch.tensor(unit * 2.0 ** -10)) + work[mine], "new")
            codes[slots[mine]] = got[slots[mine]]
            old = slice(k * block, k * block + first)
            if byte > low and first > 0:
                rose += 1
                codes[old] = (was[old].view(R.E4M3).double() * 2.0 ** (low - byte)).float().to(R.E4M3).view(torch.uint8)
        same = codes.view(R.E4M3).float() == got.view(R.E4M3).float()  # (0 and -0 are the same number)
        assert bool(same.all()) and torch.equal(scales, got_s)
        lens += np.array(n_new)
    assert rose >= 2 or block == 2  # (some block did rise)


@pytest.mark.parametrize("block, n_new", [(64, [9000, 1, 8000, 40, 9001]), (32, [13000] + [31] * 40), (4, [13001, 5])])
def test_append_many_runs(block, n_new):
    """Enough tokens that a workgroup looks for runs among many."""
    page, N = 64, sum(n_new)
    cols = -(-max(n_new) // page)
    P = sum(-(-n // page) for n in n_new)
    ids, table = np.random.default_rng(block).permutation(P), np.zeros((len(n_new), cols), np.int64)
    at = 0
    for b, n in enumerate(n_new):
        k = -(-n // page)
        table[b, :k] = ids[at:at + k]
        at += k
    seq = np.repeat(np.arange(len(n_new)), n_new)
    tok = np.concatenate([np.arange(n) for n in n_new])
    slots = table[seq, tok // page] * page + tok % page
    c, pe = bf16_randn((N, C), 1, 2.0), bf16_randn((N, PE), 2, 2.0)
    pool, scale = fresh(P, page, 8, block)
    ops.latent_rope_append(c.to(DEV), pe.to(DEV), torch.zeros((N, 1, PE), dtype=torch.bfloat16, device=DEV),
                           torch.zeros(N, dtype=torch.int32, device=DEV), torch.ones(32, device=DEV), ints(slots),
                           pool, scale)  # (position 0: nothing turns, so all of it is exact)
    x = torch.cat([c, pe], 1).float()
    group = torch.from_numpy(slots // block)
    top = torch.zeros(P * page // block).scatter_reduce_(0, group, x.abs().amax(1), "amax")
    e = torch.frexp(top / 448)
    byte = e.exponent - (e.mantissa == 0.5).int() + 127  # the least power of two >= top / 448
    used = torch.unique(group)
    got_s = scale.view(torch.uint8).cpu().view(-1)
    assert torch.equal(got_s[used].int(), byte[used])
    want = torch.ldexp(x, 127 - byte[group][:, None]).to(R.E4M3).float()
    assert torch.equal(pool.view(torch.uint8).cpu().view(-1, W)[slots].view(R.E4M3).float(), want)
    spare = torch.ones(P * page, dtype=torch.bool)
    spare[slots] = False
    assert bool((pool.view(torch.uint8).cpu().view(-1, W)[spare] == 0x31).all())


@pytest.mark.parametrize("block", (1, 32))
def test_append_odd_rows(block):
    """Rows of zeros, of very small and large values, and with an infinity or a NaN, which
    becomes NaN in its place and has no part in the scale."""
    N = 8
    c, pe = bf16_randn((N, C), 5), bf16_randn((N, PE), 6)
    c[0], pe[0] = 0, 0
    c[1], pe[1] = c[1] * 1e-38, pe[1] * 1e-38
    c[2], pe[2] = c[2] * 1e37, pe[2] * 1e37
    c[3, 7] = math.inf
    c[4, 9], pe[4, 40] = math.nan, -math.inf
    c[5], pe[5] = 448.0, 448.0
    c[6], pe[6] = 450.0, 450.0  # 448 is the largest that fits a scale of 1
    c[7] = math.nan
    slots = np.arange(N) * block  # a block each
    pool, scale = fresh(N * max(1, block // 32), 32, 8, block)
    ops.latent_rope_append(c.to(DEV), pe.to(DEV), torch.zeros((N, 1, PE), dtype=torch.bfloat16, device=DEV),
                           torch.zeros(N, dtype=torch.int32, device=DEV), torch.ones(32, device=DEV), ints(slots),
                           pool, scale)
    x = torch.cat([c, pe], 1).double()
    got = pool.view(torch.uint8).cpu().view(-1, W)[slots].view(R.E4M3).double()
    byte = scale.view(torch.uint8).cpu().view(-1)[slots // block].long()
    # (position 0: a pair with an infinity or a NaN is that in both columns; the others do not turn)
    gone = ~x.isfinite()
    gone[4, C + 8] = True  # -inf's partner: -inf * 1 beside x * 0
    for i in range(N):
        fine = x[i][x[i].isfinite()]
        want = L.exponent(float(fine.abs().max())) + 127 if i != 4 else int(byte[4])
        assert int(byte[i]) == want, i
        assert torch.equal(got[i].isnan(), gone[i]) or i == 4, i
        ok = ~gone[i]
        codes = (x[i] * 2.0 ** (127 - int(byte[i]))).float().to(R.E4M3).double()
        assert torch.equal(got[i][ok], codes[ok]), i
    assert bool(got[4][9].isnan()) and bool(got[4][C + 40].isnan()) and int(got[4].isnan().sum()) <= 3


def test_append_far_positions_and_large_squares():
    """Positions to 2^30 and below 0 (the angle is reduced in 64 bits), and rows whose squares
    leave nothing beside eps, or are large."""
    N = 40
    c, pe, q_pe, pos, inv = inputs(N, 2, 3)
    pos = pos * 26000
    pos[:3] = torch.tensor([0, -1, -(1 << 30)], dtype=torch.int32)
    c[5], c[6] = c[5] * 1e-6, c[6] * 1e15
    c[7] = 0
    weight = (1 + 0.2 * bf16_randn((C,), 4).float()).to(torch.bfloat16)
    pool, scale = fresh(2, 32, 16)
    q = ops.latent_rope_append(*on_gpu(c, pe, q_pe), pos.to(DEV), inv.to(DEV), ints(np.arange(N)), pool, None,
                               weight.to(DEV), 1e-6)
    check_q(q, q_pe, pos, inv, False, 1.0)
    x, work = L.latents(c, pe, pos, inv, False, 1.0, weight, 1e-6)
    R.check(pool.view(-1, W)[:N], x, x.abs() * 2.0 ** -8 + work, "latent")


# ---------------------------------------------------------------------------
# reading back


@pytest.mark.parametrize("bits, block", [(16, 1), (8, 1), (8, 16), (8, 64)])
@pytest.mark.parametrize("lens, start, count", [
    ([1], [0], [1]), ([200, 0, 65, 64], [3, 0, 64, 0], [190, 0, 1, 64]), ([40] * 300, [7] * 300, [33] * 300),
    ([64, 64, 1], [0, 64, 0], [0, 0, 0]), ([5000], [100], [4800])])
def test_gather(bits, block, lens, start, count):
    page = 64
    table, P, cpu = L.pools(lens, page, bits, block, len(lens))
    pool, scale = dev(cpu)
    cu = np.concatenate([[0], np.cumsum(count)])
    n = int(cu[-1])
    want = L.gather(cpu, table, start, cu, n, page, block)
    c, pe = ops.latent_gather(pool, ints(table), ints(cu), n, ints(start), scale)
    assert torch.equal(c.cpu(), want[:, :C]) and torch.equal(pe.cpu(), want[:, C:])
    # parts of one tensor, with rows before and behind, which stay
    rows = torch.full((n + 7, W), 5.0, dtype=torch.bfloat16, device=DEV)
    ops.latent_gather(pool, ints(table), ints(cu + 4), n + 7, ints(start), scale, rows[:, :C], rows[:, C:])
    assert torch.equal(rows[4:n + 4].cpu(), want) and bool((rows[:4] == 5).all()) and bool((rows[n + 4:] == 5).all())


@pytest.mark.parametrize("bits", (16, 8))
def test_gather_bad_pages_and_ranges(bits):
    lens, page = [100, 70, 40], 32
    table, P, cpu = L.pools(lens, page, bits, 1, 3)
    pool, scale = dev(cpu)
    table[0, 1], table[1, 0], table[2, 1] = P, -5, 1 << 30
    start, cu = [30, -2, 5], np.array([0, 40, 50, 200])
    want = L.gather(cpu, table, start, cu, 200, page, 1)
    assert bool(want[:2].isfinite().all()) and bool(want[2:34].isnan().all()) and bool(want[150:].isnan().all())
    c, pe = ops.latent_gather(pool, ints(table), ints(cu), 200, ints(start), scale)
    got = torch.cat([c, pe], 1).cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~want.isnan()], want[~want.isnan()])
    zero = ops.latent_gather(pool, ints(table), ints(cu[:4]), 20, None, scale)[0]  # rows past n_rows are no rows
    assert zero.shape == (20, C)


def test_gather_nan_scale():
    table, P, (pool, scale) = L.pools([40], 32, 8, 8, 5)
    scale.view(torch.uint8)[int(table[0, 0]), 2] = 255  # tokens 16 .. 23
    c, pe = ops.latent_gather(pool.to(DEV), ints(table), ints([0, 40]), 40, None, scale.to(DEV))
    bad = torch.zeros(40, dtype=torch.bool)
    bad[16:24] = True
    assert torch.equal(c.isnan().all(1).cpu(), bad) and torch.equal(pe.isnan().any(1).cpu(), bad)


def test_gather_every_code_at_every_scale():
    """All 256 codes under the scales 2^-126 to 2^127: the product to the nearest bf16, which
    it is but where it falls below 2^-133 or leaves the range."""
    page, n = 32, 254
    table, P, (pool, sc) = L.pools([n], page, 8, 1, 4)
    codes = (torch.arange(n)[:, None] * 37 + torch.arange(W)[None]).to(torch.uint8)
    for t in range(n):
        pid, off = int(table[0, t // page]), t % page
        pool.view(torch.uint8)[pid, off] = codes[t]
        sc.view(torch.uint8)[pid, off] = t + 1
    c, pe = ops.latent_gather(pool.to(DEV), ints(table), ints([0, n]), n, latent_scale=sc.to(DEV))
    want = (codes.view(R.E4M3).double() * 2.0 ** (torch.arange(n).double()[:, None] - 126)).float().to(torch.bfloat16)
    got = torch.cat([c, pe], 1).cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    low = codes[0].view(R.E4M3).double().nan_to_num(0.0) * 2.0 ** -126
    assert bool((want[0].double().nan_to_num(0.0) != low).any())  # (so it is rounded there)
    assert torch.equal(want[2:100].double().nan_to_num(0.0),
                       (codes.view(R.E4M3).double() * 2.0 ** (torch.arange(n).double()[:, None] - 126))[2:100].nan_to_num(0.0))


# ---------------------------------------------------------------------------
# attention


def queries(N, H, seed, sigma=1.0):
    return bf16_randn((N, H, C), seed, sigma), bf16_randn((N, H, PE), seed + 1, sigma)


SCALE = 192 ** -0.5


@pytest.mark.parametrize("H, page, block, lens, splits", [
    (16, 64, 1, [1], 0), (16, 64, 1, [31, 32, 33, 0, 64, 65], 0), (128, 64, 64, [200, 1, 7], 0), (1, 32, 16, [99], 1),
    (20, 96, 32, [300, 17], 7), (5, 64, 2, [129, 500], 4), (64, 64, 1, [70, 71, 72], 0), (130, 32, 1, [33, 1], 3),
    (300, 32, 1, [65], 0), (32, 64, 8, [257, 5], 6), (16, 64, 1, [3000], 256), (16, 64, 1, [40] * 70, 0),
    (8, 32, 1, [5] * 300, 0), (33, 128, 128, [1500, 0, 3, 900], 17), (16, 32, 32, [2000, 300, 1, 64], 0)])
def test_decode8(H, page, block, lens, splits):
    table, P, cpu = L.pools(lens, page, 8, block, H + len(lens))
    qn, qp = queries(len(lens), H, 9)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, None, page, block, SCALE, pieces=splits != 1)
    args = (qn.to(DEV), qp.to(DEV), *dev(cpu), ints(table), ints(lens), SCALE, max(lens), splits)
    out, lse = ops.mla8_decode_partial(*args)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    o16, l16 = ops.mla8_decode_full(*args)
    R.check(o16, want_o, tol_o + want_o.abs() * 2.0 ** -8, "bf16 out")
    R.check(l16, want_l, tol_l, "lse")
    again, _ = ops.mla8_decode_partial(*args)
    assert torch.equal(again, out)


def test_decode8_bad_pages_and_lengths():
    lens, page = [100, 70, 40, 0, 64], 32
    table, P, cpu = L.pools(lens, page, 8, 1, 21)
    pool, scale = dev(cpu)
    qn, qp = queries(5, 16, 2)
    want = L.attention(qn, qp, cpu, table, lens, None, page, 1, 0.125)
    table[0, 3] = P         # reached
    table[1, 0] = -5        # reached
    table[2, 2:] = 1 << 30  # not reached by 40 tokens
    lens[4] = page * table.shape[1] + 1  # past the row's capacity
    for fn in (ops.mla8_decode_partial, ops.mla8_decode_full):
        for splits in (1, 5, 0):
            out, lse = fn(qn.to(DEV), qp.to(DEV), pool, scale, ints(table), ints(lens), 0.125, 100, splits)
            assert bool(out[[0, 1, 4]].isnan().all()) and bool(lse[[0, 1, 4]].isnan().all())
            half = 2.0 ** -8 if out.dtype == torch.bfloat16 else 0.0
            R.check(out[2:4], want[0][2:4], want[2][2:4] + want[0][2:4].abs() * half, "fine ones")
            R.check(lse[2:4], want[1][2:4], want[3][2:4], "fine ones")
    out, lse = ops.mla8_decode_partial(qn.to(DEV), qp.to(DEV), pool, scale, ints(table), ints([-1] * 5), 0.125, 100)
    assert bool(out.isnan().all()) and bool(lse.isnan().all())


def test_decode8_scales_and_queries_of_all_sizes():
    """Token scales over a wide range, a NaN scale, and query rows whose columns differ by
    many powers of two, or hold an infinity."""
    page, n = 32, 40
    table, P, (pool, scale) = L.pools([n], page, 8, 1, 3)
    sb = scale.view(torch.uint8)
    rows = [(int(table[0, t // page]), t % page) for t in range(n)]
    for i, (p, o) in enumerate(rows):
        sb[p, o] = [90, 100, 110, 119, 121][i % 5]
    qn, qp = queries(1, 20, 4)
    qn[0, 3] *= 1e-30
    qn[0, 4, 7], qn[0, 5, 9] = 3e4, 1e6
    qn[0, 6], qp[0, 6] = 0, 0
    qn[0, 7, :100] *= 2.0 ** -18
    want = L.attention(qn, qp, (pool, scale), table, [n], None, page, 1, 0.1)

    def run(q=qn):
        return ops.mla8_decode_partial(q.to(DEV), qp.to(DEV), pool.to(DEV), scale.to(DEV), ints(table), ints([n]),
                                       0.1, n)

    out, lse = run()
    R.check(out, want[0], want[2], "out")
    R.check(lse, want[1], want[3], "lse")
    bad = qn.clone()
    bad[0, 2, 5], bad[0, 8, 500] = math.inf, math.nan
    got, got_l = run(bad)
    gone = torch.zeros(20, dtype=torch.bool)
    gone[[2, 8]] = True
    assert torch.equal(got[0].isnan().all(-1).cpu(), gone) and torch.equal(got[0].isnan().any(-1).cpu(), gone)
    assert torch.equal(got[0, ~gone], out[0, ~gone]) and torch.equal(got_l[0, ~gone], lse[0, ~gone])
    sb[rows[33]] = 255
    assert bool(run()[0].isnan().all()) and bool(run()[1].isnan().all())


def prompt_on(qn, qp, cpu, table, lens, new, scale, max_len=None, **kw):
    pool, sc = dev(cpu)
    return ops.mla_prompt(qn.to(DEV), qp.to(DEV), pool, ints(table), ints(lens),
                          ints(np.concatenate([[0], np.cumsum(new)])), scale, max_len or max(lens),
                          latent_scale=sc, out_dtype=kw.pop("out_dtype", torch.float32), **kw)


@pytest.mark.parametrize("bits, block", [(16, 1), (8, 1), (8, 32)])
@pytest.mark.parametrize("H, page, lens, new, splits", [
    (1, 32, [1], [1], 0), (16, 64, [65, 64, 1, 33], [65, 3, 1, 32], 0), (20, 32, [300, 17, 128], [130, 0, 128], 0),
    (5, 96, [200, 0, 90], [77, 0, 1], 0), (2, 32, [150], [150], 0), (128, 64, [140], [13], 0),
    (64, 64, [100, 30], [10, 7], 0), (1, 32, [700], [333], 0), (130, 64, [50, 3], [7, 3], 0),
    (16, 64, [700], [5], 0), (16, 64, [900, 400], [3, 2], 7), (40, 64, [70, 200], [2, 9], 0), (3, 128, [500], [200], 3),
    (2, 32, [3] * 150, [2] * 150, 0), (16, 64, [10, 5], [30, 5], 0), (8, 32, [400], [5], 64)])
def test_prompt(bits, block, H, page, lens, new, splits):
    """(30 queries of a 10-token partition: the first 20 see nothing.)"""
    table, P, cpu = L.pools(lens, page, bits, block, H + len(lens))
    qn, qp = queries(sum(new), H, 9)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, new, page, block, SCALE, pieces=splits != 1)
    out, lse = prompt_on(qn, qp, cpu, table, lens, new, SCALE, n_splits=splits)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    o16, none = prompt_on(qn, qp, cpu, table, lens, new, SCALE, n_splits=splits, out_dtype=torch.bfloat16,
                          want_lse=False)
    assert none is None
    R.check(o16, want_o, tol_o + want_o.abs() * 2.0 ** -8, "bf16 out")
    again, _ = prompt_on(qn, qp, cpu, table, lens, new, SCALE, n_splits=splits)
    assert torch.equal(again, out)


@pytest.mark.parametrize("bits", (16, 8))
def test_prompt_packed_elsewhere(bits):
    """Rows before the first and behind the last sequence keep what they held, at any
    split count."""
    lens, new, page = [70, 40], [9, 40], 32
    table, P, cpu = L.pools(lens, page, bits, 1, 5)
    pool, sc = dev(cpu)
    qn, qp = queries(60, 3, 1)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, new, page, 1, 0.1, c0=4)
    for splits in (1, 2):
        out, lse = torch.full((60, 3, C), 5.0, device=DEV), torch.full((60, 3), 6.0, device=DEV)
        ops.mla_prompt(qn.to(DEV), qp.to(DEV), pool, ints(table), ints(lens), ints([4, 13, 53]), 0.1, 70,
                       latent_scale=sc, out=out, lse=lse, n_splits=splits)
        R.check(out[4:53], want_o[4:53], tol_o[4:53], "out")
        R.check(lse[4:53], want_l[4:53], tol_l[4:53], "lse")
        for x, was in ((out, 5.0), (lse, 6.0)):
            assert bool((x[:4] == was).all()) and bool((x[53:] == was).all())


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("n, H, splits", [(60, 2, 0), (150, 3, 1), (3, 2, 2), (70, 16, 1)])
@pytest.mark.parametrize("column", (5, 511, 570))
def test_prompt_nonfinite_tokens(bits, n, H, splits, column):
    """An infinity or a NaN in a token's latent reaches the rows that see it and no other."""
    T, page = 200, 64
    table, P, (pool, sc) = L.pools([T], page, bits, 1, 31)
    at = T - n // 2 - 1
    pid, off = int(table[0, at // page]), at % page
    if bits == 16:
        pool[pid, off, column] = math.inf if n == 60 else math.nan
    else:
        pool.view(torch.uint8)[pid, off, column] = 0x7f
    qn, qp = queries(n, H, 3)
    out, lse = prompt_on(qn, qp, (pool, sc), table, [T], [n], 0.125, n_splits=splits)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, (pool, sc), table, [T], [n], page, 1, 0.125, pieces=splits != 1)
    clean = at - (T - n)  # rows before it
    assert clean > 0
    R.check(out[:clean], want_o[:clean], tol_o[:clean], "rows that do not see it")
    R.check(lse[:clean], want_l[:clean], tol_l[:clean], "rows that do not see it")
    if column < C:
        assert not bool(out[clean:, :, column].isfinite().any())
    if bits == 8 or n != 60:
        assert bool(out[clean:].isnan().all()) and bool(lse[clean:].isnan().all())


@pytest.mark.parametrize("H, n", [(2, 40), (16, 20)])
def test_prompt_nan_scale(H, n):
    """A scale of NaN is a NaN of its tokens, and of the rows that see them."""
    T, page = 130, 32
    table, P, (pool, sc) = L.pools([T], page, 8, 4, 9)
    at = T - n // 2
    sc.view(torch.uint8)[int(table[0, at // page]), at % page // 4] = 255
    qn, qp = queries(n, H, 3)
    out, lse = prompt_on(qn, qp, (pool, sc), table, [T], [n], 0.125)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, (pool, sc), table, [T], [n], page, 4, 0.125)
    clean = at // 4 * 4 - (T - n)
    R.check(out[:clean], want_o[:clean], tol_o[:clean], "rows that do not see it")
    R.check(lse[:clean], want_l[:clean], tol_l[:clean], "rows that do not see it")
    assert bool(out[clean:].isnan().all()) and bool(lse[clean:].isnan().all())


@pytest.mark.parametrize("block, splits", [(1, 0), (32, 1), (8, 3)])
def test_prompt_many_tiles_over_8_bits(block, splits):
    """Prompts of many tiles a sequence, whose latents are widened in a pass of their own: NaN
    codes, NaN scales and bad pages reach the rows that see them, and lengths out of range
    their own sequence."""
    lens, new, page, H = [330, 200, 64, 40, 100], [180, 130, 0, 30, 100], 32, 20
    assert sum(new) * H >= 12 * 128 * len(new)
    table, P, (pool, sc) = L.pools(lens, page, 8, block, 41)
    place = lambda b, t: (int(table[b, t // page]), t % page)
    p, o = place(0, 250)
    pool.view(torch.uint8)[p, o, 77] = 0x7f
    p, o = place(1, 150)
    sc.view(torch.uint8)[p, o // block] = 255
    qn, qp = queries(sum(new), H, 3)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, (pool, sc), table, lens, new, page, block, 0.1, pieces=splits != 1)
    table[4, 2] = P + 1  # tokens 64 .. 95
    lens[3] = -1
    out, lse = prompt_on(qn, qp, (pool, sc), table, lens, new, 0.1, n_splits=splits)
    cu = np.concatenate([[0], np.cumsum(new)])
    seen = {0: 250 - 150, 1: 150 // block * block - 70, 3: 0, 4: 64}  # rows that see nothing odd
    for b, n in seen.items():
        fine, gone = slice(cu[b], cu[b] + n), slice(cu[b] + n, cu[b + 1])
        R.check(out[fine], want_o[fine], tol_o[fine], f"fine rows of {b}")
        R.check(lse[fine], want_l[fine], tol_l[fine], f"fine rows of {b}")
        assert bool(out[gone].isnan().all()) and bool(lse[gone].isnan().all()), b


@pytest.mark.parametrize("bits", (16, 8))
def test_prompt_scale_signs(bits):
    """A negative scale, and zero (the mean of what a row sees)."""
    lens, new, page = [90], [40], 32
    table, P, cpu = L.pools(lens, page, bits, 1, 8)
    qn, qp = queries(40, 2, 1)
    for scale in (-0.2, 0.0):
        for splits in (1, 2):
            want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, new, page, 1, scale)
            out, lse = prompt_on(qn, qp, cpu, table, lens, new, scale, n_splits=splits)
            R.check(out, want_o, tol_o, f"out at scale {scale}")
            R.check(lse, want_l, tol_l, f"lse at scale {scale}")


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("H, T, n", [(1, 300, 100), (16, 500, 3)])
def test_prompt_large_scores(bits, H, T, n):
    """Scores of hundreds, whose maximum climbs out of the first block's headroom: the
    second pass."""
    page = 32
    table, P, cpu = L.pools([T], page, bits, 1, 12, sigma=2.0)
    qn, qp = queries(n, H, 1, 4.0)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, [T], [n], page, 1, 1.0, pieces=False)
    out, lse = prompt_on(qn, qp, cpu, table, [T], [n], 1.0, n_splits=1)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("splits", (1, 3))
def test_prompt_bad_pages_and_lengths(bits, splits):
    lens, new, page = [150, 100, 64, 80, 10], [100, 5, 64, 4, 3], 32
    table, P, cpu = L.pools(lens, page, bits, 1, 77)
    N = sum(new)
    qn, qp = queries(N, 4, 2)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, new, page, 1, 0.125)
    table[0, 3] = P   # tokens 96 .. 127: seen by queries from position 96 on
    table[1, 0] = -1  # seen by every query
    table[2, 2:] = 1 << 30  # never reached
    lens[3], lens[4] = -1, page * table.shape[1] + 1
    cu = np.concatenate([[0], np.cumsum(new)])
    out, lse = prompt_on(qn, qp, cpu, table, lens, new, 0.125, max_len=150, n_splits=splits)
    first = 96 - 50  # the query at position 96
    fine = list(range(first)) + list(range(cu[2], cu[3]))
    R.check(out[fine], want_o[fine], tol_o[fine], "fine rows")
    R.check(lse[fine], want_l[fine], tol_l[fine], "fine rows")
    gone = [i for i in range(N) if i not in fine]
    assert bool(out[gone].isnan().all()) and bool(lse[gone].isnan().all())


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("T, n, H", [(2090, 3, 16), (2130, 70, 2), (4230, 2, 1), (2048, 1, 8), (4096, 5, 3)])
def test_windows_of_page_ids(bits, T, n, H):
    """One workgroup walks more than 64 blocks: its window of page ids is fetched again; a
    bad page in a later window is seen."""
    page, lens, new = 32, [T, 50], [n, 1]
    table, P, cpu = L.pools(lens, page, bits, 1, T + n)
    qn, qp = queries(n + 1, H, 2)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, new, page, 1, SCALE, pieces=False)
    out, lse = prompt_on(qn, qp, cpu, table, lens, new, SCALE, n_splits=1)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    bad = -(-(T - n) // page) - 1  # a page that every row sees
    table[0, bad] = P + 3
    out, lse = prompt_on(qn, qp, cpu, table, lens, new, SCALE, n_splits=1)
    assert bool(out[:n].isnan().all()) and bool(lse[:n].isnan().all())
    R.check(out[n:], want_o[n:], tol_o[n:], "the other sequence")


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("B, splits", [(70, 3), (70, 0), (300, 3), (300, 0), (129, 0)])
def test_many_split_sequences(bits, B, splits):
    """More sequences than a wave's lanes, split: both kernels number the pieces alike.  A few
    are long, so that they are split where the lengths decide."""
    page, H, rng = 64, 4, np.random.default_rng(B)
    lens = rng.integers(1, 60, B)
    lens[rng.permutation(B)[:4]] = (700, 1500, 333, 900)
    new = np.minimum(lens, rng.integers(0, 5, B))
    new[int(np.argmax(lens))] = 40  # (two tiles of rows)
    table, P, cpu = L.pools(lens, page, bits, 1, B)
    qn, qp = queries(int(new.sum()), H, 3)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, new, page, 1, 0.1)
    out, lse = prompt_on(qn, qp, cpu, table, lens, new, 0.1, n_splits=splits)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


@pytest.mark.parametrize("B", (1, 40, 256, 300))
def test_decode8_at_a_long_capacity(B):
    """One long sequence among short ones, with the row's capacity as max_len (a captured
    step's)."""
    H, page, cap = 8, 64, 1 << 17
    lens = [int(x) for x in np.random.default_rng(B).integers(0, 70, B)]
    lens[B // 3] = 4100
    table, P, cpu = L.pools(lens, page, 8, 64, B)
    table = np.concatenate([table, np.full((B, cap // page - table.shape[1]), -1, np.int32)], 1)
    qn, qp = queries(B, H, 4)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, None, page, 64, SCALE)
    out, lse = ops.mla8_decode_partial(qn.to(DEV), qp.to(DEV), *dev(cpu), ints(table), ints(lens), SCALE, cap)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


FAR = (1 << 17) + 64  # a max_len from which few rows over 8-bit pages run in tiles of 128


def wide_table(table, page):
    return np.concatenate([table, np.full((table.shape[0], FAR // page + 1 - table.shape[1]), -1, np.int32)], 1)


@pytest.mark.parametrize("H, block, lens, splits", [
    (1024, 1, [40, 200], 0), (65, 1, [200, 1, 7], 0), (100, 64, [31, 64, 0, 65], 3), (128, 32, [500, 33], 1), (130, 1, [140], 0),
    (128, 1, [2090], 1), (72, 64, [4200, 3], 1)])
def test_decode8_tiles_of_128_rows(H, block, lens, splits):
    page = 64
    table, P, cpu = L.pools(lens, page, 8, block, H + len(lens))
    qn, qp = queries(len(lens), H, 9)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, None, page, block, SCALE, pieces=splits != 1)
    args = (qn.to(DEV), qp.to(DEV), *dev(cpu), ints(wide_table(table, page)), ints(lens), SCALE, FAR, splits)
    out, lse = ops.mla8_decode_partial(*args)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    o16, l16 = ops.mla8_decode_full(*args)
    R.check(o16, want_o, tol_o + want_o.abs() * 2.0 ** -8, "bf16 out")
    R.check(l16, want_l, tol_l, "lse")


@pytest.mark.parametrize("H, lens, new, scale, sigma, what", [
    (16, [300, 90], [7, 5], SCALE, 1.0, None), (20, [200], [4], -0.1, 1.0, None), (2, [90], [40], 0.0, 1.0, None),
    (1, [300], [100], 1.0, 4.0, None), (16, [400], [6], 0.125, 1.0, "token"), (2, [200], [60], 0.125, 1.0, "token"),
    (16, [200], [6], 0.125, 1.0, "scale"), (2, [2130], [60], SCALE, 1.0, "page")])
def test_prompt_tiles_of_128_rows_over_8_bits(H, lens, new, scale, sigma, what):
    """Scale signs, scores that climb out of the first block's headroom, NaN tokens and scales,
    a bad page in a later window of ids."""
    page, block, T, n = 32, 4, lens[0], new[0]
    splits = 1 if what == "page" or sigma > 1 else 0
    table, P, (pool, sc) = L.pools(lens, page, 8, block, 12, sigma=max(sigma / 2, 1.0))
    qn, qp = queries(sum(new), H, 1, sigma)
    at = {"token": T - n // 2 - 1, "scale": (T - 1) // block * block, "page": 2090 // page * page}.get(what, T)
    pid, off = int(table[0, min(at, T - 1) // page]), at % page
    if what == "token":
        pool.view(torch.uint8)[pid, off, 300] = 0x7f
    elif what == "scale":
        sc.view(torch.uint8)[pid, off // block] = 255
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, (pool, sc), table, lens, new, page, block, scale,
                                               pieces=splits != 1)
    if what == "page":
        table[0, at // page] = P
    out, lse = prompt_on(qn, qp, (pool, sc), wide_table(table, page), lens, new, scale, max_len=FAR, n_splits=splits)
    clean = np.arange(sum(new))
    clean = clean[(clean >= n) | (clean + T - n < at)]
    assert (what is None) == (len(clean) == sum(new)) and len(clean) > 0
    R.check(out[clean], want_o[clean], tol_o[clean], "out")
    R.check(lse[clean], want_l[clean], tol_l[clean], "lse")
    gone = np.setdiff1d(np.arange(sum(new)), clean)
    assert bool(out[gone].isnan().all()) and bool(lse[gone].isnan().all())


@pytest.mark.parametrize("bits", (16, 8))
def test_pools_past_4_gib(bits):
    """The same pages at the far end of a pool of more than 2^32 bytes: the same bits."""
    page, lens, new, block = 64, [200, 90], [40, 3], 32
    table, P, cpu = L.pools(lens, page, bits, block, 77)
    small = dev(cpu)
    Pb = 120000 * 16 // bits
    shift = Pb - P
    far = np.where(table >= 0, table + shift, table).astype(np.int32)
    big = [None if t is None else torch.zeros((Pb,) + t.shape[1:], dtype=torch.uint8, device=DEV).view(t.dtype)
           if t.element_size() == 1 else torch.zeros((Pb,) + t.shape[1:], dtype=t.dtype, device=DEV) for t in small]
    assert big[0].numel() * big[0].element_size() > 1 << 32
    N = 50
    c, pe, q_pe, pos, inv = (t.to(DEV) for t in inputs(N, 4, 5))
    slots = np.array([int(table[0, t // page]) * page + t % page for t in range(100, 100 + N)])
    raw = lambda t: t.view(torch.uint8)
    for a, b in zip(big, small):
        if a is not None:
            raw(a)[shift:] = raw(b)
    for pools, s in ((small, slots), (big, slots + shift * page)):
        ops.latent_rope_append(c, pe, q_pe, pos, inv, ints(s), *pools)
    for a, b in zip(big, small):
        if a is not None:
            assert torch.equal(raw(a)[shift:], raw(b)) and not bool(raw(a)[:shift].any())
    qn, qp = (t.to(DEV) for t in queries(43, 4, 6))
    calls = [lambda p, t: ops.mla_prompt(qn, qp, p[0], ints(t), ints(lens), ints([0, 40, 43]), 0.1, 200,
                                         latent_scale=p[1]),
             lambda p, t: ops.latent_gather(p[0], ints(t), ints([0, 100, 150]), 150, ints([20, 30]), p[1])]
    if bits == 8:
        calls.append(lambda p, t: ops.mla8_decode_partial(qn[:2], qp[:2], *p, ints(t), ints(lens), 0.1, 200))
    for call in calls:
        for x, y in zip(call(small, table), call(big, far)):
            assert bool(x.isfinite().all()) and torch.equal(x, y)


def test_refused_tensors():
    t = torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    x = torch.zeros((4, W), dtype=torch.bfloat16, device=DEV)
    c, pe = x[:, :C], x[:, C:]
    q = torch.zeros((4, 2, PE), dtype=torch.bfloat16, device=DEV)
    qn = torch.zeros((4, 2, C), dtype=torch.bfloat16, device=DEV)
    pos, inv = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(32, device=DEV)
    pool = torch.zeros((3, 32, W), dtype=torch.bfloat16, device=DEV)
    p8, s8 = fresh(3, 32, 8, 4)
    cu = torch.zeros(3, dtype=torch.int32, device=DEV)
    for kw, err, says in (
            (dict(c=x), ValueError, "c must"), (dict(pe=pe.float()), TypeError, "pe"), (dict(q_pe=qn), ValueError, "q_pe"),
            (dict(positions=pos[:3]), ValueError, "positions"), (dict(inv_freq=inv[:31]), ValueError, "inv_freq"),
            (dict(slots=pos.long()), TypeError, "slots"), (dict(latent_pages=pool[..., :C].contiguous()), ValueError, "576"),
            (dict(latent_scale=s8), TypeError, "float8_e4m3fn"), (dict(latent_pages=p8), TypeError, "bfloat16"),
            (dict(latent_pages=p8, latent_scale=s8[:2]), ValueError, "latent_scale"),
            (dict(latent_pages=p8, latent_scale=s8[:, :3].contiguous()), ValueError, "latent_scale"),
            (dict(norm_weight=inv), ValueError, "norm_weight"), (dict(norm_weight=x[0, :C].half()), TypeError, "norm_weight"),
            (dict(eps=-1.0, norm_weight=x[0, :C]), ops.WsError, "eps"), (dict(q_out=q[:3]), ValueError, "q_out"),
            (dict(c=torch.zeros((C, 4), dtype=torch.bfloat16, device=DEV).t()), ValueError, "stride")):
        with pytest.raises(err, match=says):
            ops.latent_rope_append(**{**dict(c=c, pe=pe, q_pe=q, positions=pos, inv_freq=inv, slots=pos,
                                             latent_pages=pool), **kw})
    for kw, err, says in (
            (dict(cu_rows=n), ValueError, "cu_rows"), (dict(start=cu), ValueError, "start"), (dict(n_rows=-1), ValueError, "n_rows"),
            (dict(c_out=x), ValueError, "c_out"), (dict(page_table=t.long()), TypeError, "page_table")):
        with pytest.raises(err, match=says):
            ops.latent_gather(**{**dict(latent_pages=pool, page_table=t, cu_rows=cu, n_rows=4), **kw})
    for kw, err, says in (
            (dict(latent_pages=pool), TypeError, "float8_e4m3fn"), (dict(latent_scale=None), TypeError, "latent_scale"),
            (dict(gpu_len=cu), ValueError, "batch"), (dict(q_pe=q[:2, :1].contiguous()), ValueError, "q_pe"),
            (dict(q_nope=qn[:2].float()), TypeError, "q_nope"), (dict(out_bf16=qn[:2].float()), TypeError, "out_bf16"),
            (dict(lse=inv.view(16, 2)), ValueError, "lse"), (dict(n_splits=257), ops.WsError, "n_splits"),
            (dict(max_len=97), ops.WsError, "paging"), (dict(scale=math.nan), ops.WsError, "finite")):
        with pytest.raises(err, match=says):
            ops.mla8_decode_full(**{**dict(q_nope=qn[:2], q_pe=q[:2], latent_pages=p8, latent_scale=s8, page_table=t,
                                           gpu_len=n, scale=1.0, max_len=3), **kw})
    for kw, err, says in (
            (dict(cu_new=n), ValueError, "cu_new"), (dict(out_dtype=torch.float16), TypeError, "out_dtype"),
            (dict(out=qn[:3]), ValueError, "out"), (dict(kv_len=cu), ValueError, "kv_len"),
            (dict(latent_scale=s8), TypeError, "float8_e4m3fn")):
        with pytest.raises(err, match=says):
            ops.mla_prompt(**{**dict(q_nope=qn, q_pe=q, latent_pages=pool, page_table=t, kv_len=n, cu_new=cu, scale=1.0,
                                     max_len=3), **kw})


@pytest.mark.parametrize("bits, far", [(16, False), (8, False), (8, True)])
@pytest.mark.parametrize("n, H, splits", [(3, 4, 1), (40, 4, 1), (3, 4, 2)])
def test_prompt_first_blocks_of_infinite_scores(bits, far, n, H, splits):
    """Every score of the first 40 tokens is -inf (over 8-bit pages by a product past fp32's
    range), the others' lie far below 0: the first block gives the softmax no reference, and
    the others are what counts."""
    T, page, lead, scale = 150, 64, 40, 0.1
    table, P, (pool, sc) = L.pools([T], page, bits, 1, 23)
    raw = pool if bits == 16 else pool.view(torch.uint8)
    for t in range(T):
        p, o = int(table[0, t // page]), t % page
        if bits == 16:
            raw[p, o, C:C + 8] = math.inf if t < lead else 64.0
        elif t < lead:
            raw[p, o] = 0
            raw[p, o, C:C + 8] = 0x77  # 240, at a scale of 2^120
            sc.view(torch.uint8)[p, o] = 247
        else:
            raw[p, o, C:C + 8] = 0x78  # 256
            sc.view(torch.uint8)[p, o] = 125
    qn, qp = queries(n, H, 5)
    qp[..., :8] = -16.0
    rows = L.rows_of(pool, sc, table[0], T, page)
    vis = [T - n + i + 1 - lead for i in range(n)]
    want_o, want_l, tol_o, tol_l = L.attend(torch.cat([qn, qp], -1).double(), rows[lead:], vis, scale, splits != 1)
    assert float(want_l.max()) < -300
    out, lse = prompt_on(qn, qp, (pool, sc), wide_table(table, page) if far else table, [T], [n], scale,
                         max_len=FAR if far else None, n_splits=splits)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


def without_token(q, rows, at, vis, scale, pieces):
    """attend() of queries for which token `at` has the weight 0: that token left out."""
    kept = torch.cat([rows[:at], rows[at + 1:]])
    return L.attend(q, kept, [v - (v > at) for v in vis], scale, pieces)


@pytest.mark.parametrize("H, n, splits", [(2, 60, 1), (2, 60, 2), (1, 100, 0), (16, 20, 1), (16, 4, 0)])
@pytest.mark.parametrize("column, value", [(5, math.inf), (511, -math.inf), (570, math.inf), (570, -math.inf)])
@pytest.mark.parametrize("place", ("seen whole", "masked early", "masked", "last"))
def test_prompt_infinite_scores(H, n, splits, column, value, place):
    """An infinity in a token's latent, under queries whose score of it is +inf in some rows
    and -inf in others.  -inf has the weight 0, wherever the row's tile ends: the row is what
    it is without the token, but for the token's own column (0 * inf).  +inf leaves nothing of
    the row, and rows that do not see the token are as if it were not there."""
    T, page = 200, 64
    at = {"seen whole": 20, "masked early": T - n + 1, "masked": T - n // 2 - 1, "last": T - 2}[place]
    table, P, (pool, _) = L.pools([T], page, 16, 1, 17)
    rows = L.rows_of(pool, None, table[0], T, page)
    pool[int(table[0, at // page]), at % page, column] = value
    qn, qp = queries(n, H, 5)
    sign = torch.where(torch.rand((n, H), generator=torch.Generator().manual_seed(n)) < 0.6, -1.0, 1.0)
    sign.view(-1)[-2:] = torch.tensor([1.0, -1.0])  # (both, whatever sees the token)
    size = sign * (1 if value > 0 else -1)  # score: sign * inf
    (qn if column < C else qp)[..., column if column < C else column - C] = size.to(torch.bfloat16)
    out, lse = prompt_on(qn, qp, (pool, None), table, [T], [n], 0.125, n_splits=splits)
    out, lse = out.cpu(), lse.cpu()
    q = torch.cat([qn, qp], -1).double()
    vis = [T - n + i + 1 for i in range(n)]
    sees = torch.tensor(vis)[:, None] > at
    want_o, want_l, tol_o, tol_l = without_token(q, rows, at, vis, 0.125, splits != 1)
    gone, zero = sees & (sign > 0), sees & (sign < 0)
    assert bool(gone.any()) and bool(zero.any())
    assert bool(out[gone].isnan().all()) and not bool(lse[gone].isfinite().any())
    if column < C:
        assert bool(out[zero][:, column].isnan().all())
        out[..., column][zero] = want_o[..., column][zero].float()
    fine = ~gone
    R.check(out[fine], want_o[fine], tol_o[fine], "out")
    R.check(lse[fine], want_l[fine], tol_l[fine], "lse")


def test_prompt_copy_of_idle_sequences():
    """Prompts of many tiles over 8-bit pages beside sequences without new tokens: the
    widened copy takes the latents of those that have some, and no others."""
    lens, new, page, H = [300, 5000, 290, 400, 0], [200, 0, 150, 1, 0], 32, 24
    N, B, max_len = sum(new), len(lens), max(lens)
    assert N * H >= 12 * 128 * B
    table, P, cpu = L.pools(lens, page, 8, 4, 6)
    pool, sc = dev(cpu)
    qn, qp = queries(N, H, 3)
    dqn, dqp, t, l, cu = qn.to(DEV), qp.to(DEV), ints(table), ints(lens), ints(np.concatenate([[0], np.cumsum(new)]))
    _, size = ops.mla_prompt_plan(N, B, H, max_len, fp8=True)
    pad = -(-max_len // 32) * 32
    ws = torch.full((size,), 0xa5, dtype=torch.uint8, device=DEV)
    out, lse = torch.empty((N, H, C), device=DEV), torch.empty((N, H), device=DEV)
    assert ops.lib().ws_mla_prompt(
        dqn.data_ptr(), dqp.data_ptr(), pool.data_ptr(), sc.data_ptr(), t.data_ptr(), l.data_ptr(), cu.data_ptr(), N, B, H,
        page, table.shape[1], P, 4, max_len, 0, SCALE, None, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), size,
        torch.cuda.current_stream().cuda_stream) == 0
    rows = ws[size - B * pad * 2 * W:].view(B, pad, 2 * W).cpu()
    for b, n in enumerate(new):
        want = L.rows_of(*cpu, table[b], lens[b], page, 4)
        if n:
            assert torch.equal(rows[b, :lens[b]].contiguous().view(torch.bfloat16).double(), want), b
            assert bool((rows[b, lens[b]:] == 0xa5).all()), b
        else:
            assert bool((rows[b] == 0xa5).all()), f"sequence {b} has no rows that read its copy"
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, new, page, 4, SCALE)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


def test_max_len_picks_the_kernel_not_the_result():
    """The same call at its longest sequence's length and at the row's capacity (a captured
    step's): other kernels run, and each result is within its bounds."""
    page, cap = 64, 1 << 17
    wide = lambda t: np.concatenate([t, np.full((t.shape[0], cap // page - t.shape[1]), -1, np.int32)], 1)
    lens, H = [300, 70], 100  # (more than 64 rows a sequence)
    table, P, cpu = L.pools(lens, page, 8, 1, 3)
    qn, qp = queries(2, H, 9)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, None, page, 1, SCALE)
    for max_len in (300, cap):
        out, lse = ops.mla8_decode_partial(qn.to(DEV), qp.to(DEV), *dev(cpu), ints(wide(table)), ints(lens), SCALE, max_len)
        R.check(out, want_o, tol_o, f"decode at {max_len}")
        R.check(lse, want_l, tol_l, f"decode's lse at {max_len}")
    lens, new, H = [300, 200], [180, 150], 20  # (12 tiles of rows a sequence: a widened copy, where it fits)
    table, P, cpu = L.pools(lens, page, 8, 32, 4)
    N = sum(new)
    copied = [ops.mla_prompt_plan(N, 2, H, m, 1, fp8=True)[1] > ops.mla_prompt_plan(N, 2, H, m, 1)[1] for m in (300, cap)]
    assert copied == [True, False]
    qn, qp = queries(N, H, 9)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, new, page, 32, SCALE)
    for max_len in (300, cap):
        out, lse = prompt_on(qn, qp, cpu, wide(table), lens, new, SCALE, max_len=max_len)
        R.check(out, want_o, tol_o, f"prompt at {max_len}")
        R.check(lse, want_l, tol_l, f"prompt's lse at {max_len}")


@pytest.mark.parametrize("bits, block", [(16, 1), (8, 1), (8, 64)])
@pytest.mark.parametrize("H, chunk", [(16, 130), (5, 300)])
def test_one_chunk_beside_single_tokens(bits, block, H, chunk):
    """A step of continuous batching: one chunk among single tokens and sequences without any,
    every row of it."""
    page, rng = 64, np.random.default_rng(chunk)
    lens, new = rng.integers(1, 700, 30), np.ones(30, np.int64)
    lens[11], new[11] = chunk + 333, chunk
    new[[4, 29]] = 0
    table, P, cpu = L.pools(lens, page, bits, block, 8)
    qn, qp = queries(int(new.sum()), H, 9)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, new, page, block, SCALE)
    out, lse = prompt_on(qn, qp, cpu, table, lens, new, SCALE, max_len=int(max(lens)))
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


@pytest.mark.parametrize("bits, B, H, n", [(8, 8, 16, 4), (8, 12, 16, 3), (16, 20, 4, 7), (8, 16, 16, 2)])
def test_prompt_joins_of_few_tiles(bits, B, H, n):
    """Drafted tokens whose rows fill their tiles, split far: the pieces of a row are joined by a
    workgroup."""
    page, rng = 64, np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(600, 3000, B)]
    table, P, cpu = L.pools(lens, page, bits, 1, B)
    qn, qp = queries(B * n, H, 9)
    want_o, want_l, tol_o, tol_l = L.attention(qn, qp, cpu, table, lens, [n] * B, page, 1, SCALE)
    out, lse = prompt_on(qn, qp, cpu, table, lens, [n] * B, SCALE)
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
    again, _ = prompt_on(qn, qp, cpu, table, lens, [n] * B, SCALE)
    assert torch.equal(again, out)


@pytest.mark.parametrize("H, n, splits", [(2, 60, 1), (1, 100, 2), (16, 4, 1)])
@pytest.mark.parametrize("column", (5, 570))
def test_prompt_infinite_scores_in_two_passes(H, n, splits, column):
    """The same with scores that climb out of the first block's headroom: the second pass
    cleans and marks its tiles anew."""
    T, page = 300, 32
    table, P, (pool, _) = L.pools([T], page, 16, 1, 12, sigma=2.0)
    rows = L.rows_of(pool, None, table[0], T, page)
    qn, qp = queries(n, H, 1, 4.0)
    at = T - n // 2 - 1
    pool[int(table[0, at // page]), at % page, column] = -math.inf
    (qn if column < C else qp)[..., column % C] = 1.0  # every score of it is -inf
    out, lse = prompt_on(qn, qp, (pool, None), table, [T], [n], 1.0, n_splits=splits)
    out, lse = out.cpu(), lse.cpu()
    q, vis = torch.cat([qn, qp], -1).double(), [T - n + i + 1 for i in range(n)]
    want_o, want_l, tol_o, tol_l = without_token(q, rows, at, vis, 1.0, splits != 1)
    if column < C:
        sees = torch.tensor(vis) > at
        assert bool(out[sees][..., column].isnan().all())
        out[sees, :, column] = want_o[sees, :, column].float()
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")
