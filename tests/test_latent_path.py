"""The latent path's operators without a GPU: what the library refuses on the host (no
kernel is launched), the plans' arithmetic, and the plain oracle's own properties."""
import ctypes
import math

import numpy as np
import pytest
import torch

from scope_amd import ops
from tests import latent_oracle as L
from tests import request_oracle as R
from tests.helpers import bf16_randn

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: rejected before launch
ODD = ctypes.c_void_p(0x1008)


def err():
    return ops.lib().ws_last_error().decode()


def append(**kw):
    a = dict(c=FAKE, cs=576, pe=FAKE, ps=576, q=FAKE, qs=1024, qh=64, pos=FAKE, inv=FAKE, adjacent=0, factor=1.0,
             weight=None, f32=0, eps=1e-6, slots=FAKE, q_out=FAKE, pages=FAKE, scale=None, block=0, N=3, H=16, page=64,
             P=4)
    a.update(kw)
    return ops.lib().ws_latent_rope_append(*a.values(), None)


@pytest.mark.parametrize("kw, says", [
    (dict(c=None), "null"), (dict(pe=None), "null"), (dict(q=None), "null"), (dict(pos=None), "null"),
    (dict(inv=None), "null"), (dict(slots=None), "null"), (dict(q_out=None), "null"), (dict(pages=None), "null"),
    (dict(N=-1), "bad sizes"), (dict(H=0), "bad sizes"), (dict(H=1025), "bad sizes"), (dict(cs=511), "strides"),
    (dict(cs=516), "strides"), (dict(ps=60), "strides"), (dict(qh=63), "strides"), (dict(qs=1000), "strides"),
    (dict(qs=1023), "strides"), (dict(c=ODD), "aligned"), (dict(pages=ODD), "aligned"), (dict(q_out=ODD), "aligned"),
    (dict(weight=ODD), "aligned"), (dict(page=0), "paging"), (dict(P=1 << 26), "32-bit"),
    (dict(scale=FAKE, block=3), "scale_block"), (dict(scale=FAKE, block=128), "scale_block"),
    (dict(scale=FAKE, block=0), "scale_block"), (dict(scale=FAKE, block=32, page=48), "scale_block"),
    (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"),
    (dict(N=1 << 30, H=1), "launch grid")])
def test_append_refusals(kw, says):
    assert append(**kw) == -1 and says in err()


def gather(**kw):
    a = dict(pages=FAKE, scale=None, block=0, table=FAKE, start=None, cu=FAKE, c=FAKE, cs=512, pe=FAKE, ps=64, N=3, B=2,
             page=64, max_pages=4, P=4)
    a.update(kw)
    return ops.lib().ws_latent_gather(*a.values(), None)


@pytest.mark.parametrize("kw, says", [
    (dict(pages=None), "null"), (dict(table=None), "null"), (dict(cu=None), "null"), (dict(c=None), "null"),
    (dict(pe=None), "null"), (dict(N=-1), "bad sizes"), (dict(B=2049), "bad sizes"), (dict(max_pages=0), "bad sizes"),
    (dict(cs=500), "aligned"), (dict(ps=68), "aligned"), (dict(c=ODD), "aligned"), (dict(page=-1), "paging"),
    (dict(scale=FAKE, block=48), "scale_block")])
def test_gather_refusals(kw, says):
    assert gather(**kw) == -1 and says in err()


def decode8(full, **kw):
    a = dict(qn=FAKE, qp=FAKE, pages=FAKE, scale=FAKE, table=FAKE, lens=FAKE, B=1, H=16, page=64, max_pages=4, P=4,
             block=1, max_len=100, n=0, s=1.0, out=FAKE, lse=FAKE, ws=None, wsb=0)
    a.update(kw)
    fn = ops.lib().ws_mla8_decode_full if full else ops.lib().ws_mla8_decode_partial
    return fn(*a.values(), None)


@pytest.mark.parametrize("full", (True, False))
@pytest.mark.parametrize("kw, rc, says", [
    (dict(scale=None), -1, "null"), (dict(out=None), -1, "null"), (dict(lse=None), -1, "null"), (dict(qn=None), -1, "null"),
    (dict(B=2049), -1, "bad sizes"), (dict(B=-1), -1, "bad sizes"), (dict(H=0), -1, "bad sizes"), (dict(H=1025), -1, "bad sizes"),
    (dict(n=257), -1, "bad sizes"), (dict(n=-1), -1, "bad sizes"), (dict(page=48, max_len=10), -1, "paging"),
    (dict(max_len=257), -1, "paging"), (dict(P=1 << 25), -1, "31-bit"), (dict(qp=ODD), -1, "aligned"), (dict(out=ODD), -1, "aligned"),
    (dict(block=5), -1, "scale_block"), (dict(block=128), -1, "scale_block"), (dict(s=math.inf), -1, "finite"),
    (dict(s=math.nan), -1, "finite"), (dict(n=2), -3, "workspace"), (dict(n=2, ws=ctypes.c_void_p(0x1010), wsb=1 << 40), -1, "256-byte"),
    (dict(max_len=200), -3, "workspace")])
def test_decode8_refusals(full, kw, rc, says):
    assert decode8(full, **kw) == rc and says in err()


def prompt(**kw):
    a = dict(qn=FAKE, qp=FAKE, pages=FAKE, scale=None, table=FAKE, lens=FAKE, cu=FAKE, N=10, B=1, H=16, page=64,
             max_pages=4, P=4, block=0, max_len=100, n=0, s=1.0, o16=FAKE, o32=None, lse=FAKE, ws=None, wsb=0)
    a.update(kw)
    return ops.lib().ws_mla_prompt(*a.values(), None)


@pytest.mark.parametrize("kw, rc, says", [
    (dict(cu=None), -1, "null"), (dict(o16=None), -1, "null"), (dict(lens=None), -1, "null"), (dict(N=-1), -1, "bad sizes"),
    (dict(B=2049), -1, "bad sizes"), (dict(n=257), -1, "bad sizes"), (dict(page=16, max_len=10), -1, "paging"),
    (dict(max_len=257), -1, "paging"), (dict(P=1 << 26), -1, "31-bit"), (dict(qn=ODD), -1, "aligned"),
    (dict(s=math.nan), -1, "finite"), (dict(N=1 << 28), -1, "row index range"), (dict(N=1 << 26, H=1, B=1, n=256), -1, "launch grid"),
    (dict(n=2), -3, "workspace"), (dict(scale=FAKE, block=3), -1, "scale_block"), (dict(N=100, scale=FAKE, block=1), -3, "workspace")])
def test_prompt_refusals(kw, rc, says):
    assert prompt(**kw) == rc and says in err()


def test_python_layer_wants_gpu_tensors():
    i = torch.zeros((2, 3), dtype=torch.int32)
    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="on a GPU"):
        ops.latent_rope_append(x[:, 0], x[:, 0], x, i[0], torch.zeros(32), i[0], x)
    with pytest.raises(ValueError, match="on a GPU"):
        ops.latent_gather(x, i, i[0], 3)
    with pytest.raises(ValueError, match="on a GPU"):
        ops.mla8_decode_full(x, x, x, x, i, i[0], 1.0, 3)
    with pytest.raises(TypeError, match="tensor"):
        ops.mla_prompt(None, x, x, i, i[0], i[0], 1.0, 3)


def test_plans():
    pad = lambda n: -(-n // 256) * 256
    # bf16 pieces and their lse
    n, wsb = ops.mla8_plan(8, 16, 30000, 4)
    assert n == 32 and wsb == pad(32 * 16 * 4) + 32 * 16 * 512 * 2
    n, wsb = ops.mla8_plan(3, 200, 30000, 2)  # two tiles of 128 rows a sequence
    assert n == 12 and wsb == pad(12 * 128 * 4) + 12 * 128 * 512 * 2
    # one split, or no more than four blocks: none
    assert ops.mla8_plan(8, 16, 30000, 1) == (0, 0) and ops.mla8_plan(8, 16, 128) == (0, 0)
    assert ops.mla8_plan(1, 16, 129)[0] > 1 and ops.mla8_plan(0, 16, 5000, 0)[0] >= 0
    # many sequences: pieces for what can be split, not for every sequence
    assert ops.mla8_plan(2048, 128, 1 << 17)[0] <= 2 * 256 + 64
    # prompts of many tiles over 8-bit pages take a copy of their latents, up to a bound
    p16, w16 = ops.mla_prompt_plan(4000, 4, 16, 9000)
    p8, w8 = ops.mla_prompt_plan(4000, 4, 16, 9000, fp8=True)
    assert p16 == p8 and w8 == w16 + 256 + 4 * 9024 * 1152
    few = ops.mla_prompt_plan(64, 4, 16, 9000, fp8=True)
    assert few[1] < w16 and ops.mla_prompt_plan(4000, 4, 16, 1 << 17, fp8=True)[1] == w16
    with pytest.raises(ops.WsError, match="bad sizes"):
        ops.mla_prompt_plan(1, 1, 0, 100)


def test_oracle_attention_is_plain_attention():
    """The restatement beside a softmax over all scores, and its bounds above 0."""
    q, k = bf16_randn((3, 2, L.W), 1).double(), bf16_randn((40, L.W), 2).double()
    out, lse, tol_o, tol_l = L.attend(q, k, [40, 13, 0], 0.1, True)
    s = torch.einsum("nhd,td->nht", q, k) * 0.1
    assert torch.allclose(out[0], torch.softmax(s[0], -1) @ k[:, :L.C]) and torch.allclose(lse[1], torch.logsumexp(s[1, :, :13], -1))
    assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all())
    assert bool((tol_o[:2] > 0).all()) and bool((tol_l[:2] > 0).all()) and float(tol_l.max()) < 1e-2


def test_oracle_latents_and_pools():
    c, pe = bf16_randn((5, L.C), 1), bf16_randn((5, L.PE), 2)
    w = 1 + 0.1 * bf16_randn((L.C,), 3)
    x, work = L.latents(c, pe, torch.zeros(5, dtype=torch.int32), torch.ones(32), False, 1.0, w, 0.0)
    assert torch.allclose((x[:, :L.C] / w.double()).square().mean(-1), torch.ones(5, dtype=torch.float64))
    assert torch.equal(x[:, L.C:], pe.double()) and bool((work >= 0).all())  # position 0: nothing turns
    table, P, (pool, scale) = L.pools([70, 3], 32, 8, 16, 5)
    rows = L.rows_of(pool, scale, table[0], 70, 32, 16)
    assert bool(rows.isfinite().all()) and scale.shape == (P, 2)
    unit = scale.view(torch.uint8)[int(table[0, 0]), 0].double()
    top = float(rows[:16].abs().max())
    assert 208 * 2.0 ** (float(unit) - 127) <= top <= 448 * 2.0 ** (float(unit) - 127)
    got = L.gather((pool, scale), table, [60, 1], [0, 10, 12], 14, 32, 16)
    assert torch.equal(got[:10].double(), rows[60:70]) and bool((got[12:] == 5).all())


def test_exponent_rule():
    assert [L.exponent(x) for x in (448.0, 449.0, 0.0, 2.0 ** -130, 3e38, 1.75 * 2.0 ** -118)] == \
        [0, 1, -126, -126, math.ceil(math.log2(3e38 / 448)), -126]
    assert R.E8M0 == ops.E8M0 and np.isfinite(L.exponent(1e-40))


@pytest.mark.parametrize("B, H, most", [
    (1, 16, (1 << 24) - 33), (130, 16, 32 * 4032 - 1), (3, 48, 32 * ((1 << 19) // 9) - 1), (64, 128, 32 * 8191 - 1),
    (65, 128, 32 * 8065 - 1), (32, 32, 32 * 16383 - 1), (31, 32, 32 * 8456 - 1), (256, 128, 32 * 2047 - 1)])
def test_decode_fits_is_what_the_launch_takes(B, H, most):
    """The query beside the launch's own check, at the longest sequences that it takes and
    one token past them: 128 heads (and 32 to 112 from 1024 rows on) count sequences, other
    calls groups of 16 heads."""
    def launch(n):
        pages = n // 64 + 1
        return ops.lib().ws_mla_decode_partial(FAKE, FAKE, FAKE, FAKE, FAKE, B, H, 64, pages, 4, n, 0, 1.0, FAKE, FAKE,
                                               None, 0, None)
    for n, fits in ((most, True), (most + 1, False), (100, True)):
        assert ops.mla_decode_fits(B, H, n) is fits
        assert launch(n) == (-3 if fits else -1) and ("workspace" if fits else "block index range") in err()
    assert not ops.mla_decode_fits(B, H, -1)


def test_decode_fits_batches():
    assert ops.mla_decode_fits(2048, 16, 100) and not ops.mla_decode_fits(2049, 16, 100)
    assert ops.mla_decode_fits(256, 128, 100) and not ops.mla_decode_fits(257, 128, 100)
    assert not any(ops.mla_decode_fits(1, H, 100) for H in (0, -16, 8, 20, 100))
    assert ops.mla_decode_fits(0, 16, 100) and not ops.mla_decode_fits(-1, 16, 100)


@pytest.mark.parametrize("N", (1 << 30, (1 << 31) - 800, (1 << 31) - 1))
@pytest.mark.parametrize("block", (0, 1, 32))
def test_tokens_past_the_launch_grid(N, block):
    """Counts up to the largest 32-bit number are refused, not wrapped around."""
    scale = FAKE if block else None
    assert append(N=N, H=1, qs=64, scale=scale, block=block) == -1 and "launch grid" in err()
    assert gather(N=N, scale=scale, block=block) == -1 and "launch grid" in err()
