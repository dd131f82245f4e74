"""Request-path operators without a GPU: what the library refuses on the host
(no kernel is launched), the plans' arithmetic, the axis helper, and the plain
page oracle's own properties."""
import ctypes

import numpy as np
import pytest
import torch

from scope_amd import ops
from tests import request_oracle as R

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: rejected before launch
OTHER = ctypes.c_void_p(0x2000)
ODD = ctypes.c_void_p(0x1008)


def err():
    return ops.lib().ws_last_error().decode()


def extend(**kw):
    a = dict(table=FAKE, len_in=FAKE, n_new=FAKE, stack=FAKE, free_in=FAKE, base=None, len_out=OTHER,
             cu=OTHER, pos=OTHER, slots=OTHER, free_out=OTHER, B=2, max_pages=4, num_pages=8,
             stack_size=8, page=64, n=10)
    a.update(kw)
    return ops.lib().ws_pages_extend(*a.values(), None)


@pytest.mark.parametrize("kw, says", [
    (dict(table=None), "null"), (dict(free_in=None), "null"), (dict(stack=None), "null"),
    (dict(slots=None), "null"), (dict(B=-1), "bad sizes"), (dict(B=2049), "bad sizes"),
    (dict(page=0), "bad sizes"), (dict(max_pages=0), "bad sizes"),
    (dict(page=1 << 20, max_pages=1 << 11), "bad sizes"), (dict(stack_size=-1), "bad sizes"),
    (dict(num_pages=-1), "32-bit"), (dict(num_pages=1 << 26), "32-bit"), (dict(n=-1), "32-bit"),
    (dict(len_out=FAKE), "alias"), (dict(free_out=FAKE), "alias")])
def test_extend_refusals(kw, says):
    assert extend(**kw) == -1 and says in err()


@pytest.mark.parametrize("kw, says", [
    (dict(done=None), "null"), (dict(B=4000), "bad sizes"), (dict(page=-64), "bad sizes"),
    (dict(len_out=FAKE), "alias"), (dict(free_out=FAKE), "alias")])
def test_release_refusals(kw, says):
    a = dict(table=FAKE, len_in=FAKE, done=FAKE, stack=FAKE, free_in=FAKE, len_out=OTHER,
             free_out=OTHER, B=2, max_pages=4, stack_size=8, page=64)
    a.update(kw)
    assert ops.lib().ws_pages_release(*a.values(), None) == -1 and says in err()


def rope_append(**kw):
    a = dict(q=FAKE, qs=512, k=FAKE, ks=256, v=FAKE, vs=256, pos=FAKE, axes=1, inv=FAKE, axis=None,
             adjacent=0, factor=1.0, slots=FAKE, q_out=FAKE, kp=FAKE, vp=FAKE, ksc=None, vsc=None,
             N=3, Hq=4, Hkv=2, D=128, rot=128, page=64, P=4)
    a.update(kw)
    return ops.lib().ws_rope_append(*a.values(), None)


@pytest.mark.parametrize("kw, says", [
    (dict(q=None), "null"), (dict(v=None), "null"), (dict(slots=None), "null"),
    (dict(ksc=FAKE), "null"), (dict(inv=None), "null"), (dict(D=120), "bad sizes"),
    (dict(D=272, rot=16), "bad sizes"), (dict(rot=0), "bad sizes"), (dict(rot=136), "bad sizes"),
    (dict(rot=24), "bad sizes"), (dict(axes=5), "bad sizes"), (dict(axes=0), "bad sizes"),
    (dict(N=-1), "bad sizes"), (dict(Hkv=0), "bad sizes"), (dict(qs=511), "strides"),
    (dict(qs=516), "strides"), (dict(ks=100), "strides"), (dict(vs=255), "stride"),
    (dict(axis=bytes([1] + [0] * 63)), "axis"), (dict(axes=2, axis=bytes([2] * 64)), "axis"),
    (dict(q=ODD), "aligned"), (dict(kp=ODD), "aligned"), (dict(page=0), "paging"),
    (dict(P=1 << 26), "32-bit")])
def test_rope_refusals(kw, says):
    assert rope_append(**kw) == -1 and says in err()


def decode8(full=False, **kw):
    a = dict(q=FAKE, kp=FAKE, vp=FAKE, ks=FAKE, vs=FAKE, table=FAKE, lens=FAKE, B=1, Hq=32, Hkv=8,
             D=128, page=64, max_pages=4, P=4, max_len=100, n=0, scale=1.0, out=FAKE, lse=FAKE,
             ws=None, wsb=0)
    a.update(kw)
    return ops.lib().ws_gqa8_decode_partial(*a.values(), None)


@pytest.mark.parametrize("kw, rc, says", [
    (dict(ks=None), -1, "null"), (dict(out=None), -1, "null"), (dict(Hq=33), -1, "heads"),
    (dict(Hq=136), -1, "group size"), (dict(D=48), -1, "head_dim"), (dict(D=288), -1, "head_dim"),
    (dict(page=48), -1, "paging"), (dict(max_len=257), -1, "paging"), (dict(B=2049), -1, "batch"),
    (dict(n=-1), -1, "n_splits"), (dict(q=ODD), -1, "aligned"), (dict(P=1 << 24), -1, "32-bit"),
    (dict(n=16), -3, "workspace"), (dict(n=5000, ws=FAKE, wsb=1 << 40), -1, "splits")])
def test_decode8_refusals(kw, rc, says):
    assert decode8(**kw) == rc and says in err()


def prompt(**kw):
    a = dict(q=FAKE, kp=FAKE, vp=FAKE, ks=None, vs=None, table=FAKE, lens=FAKE, cu=FAKE, N=10, B=1,
             Hq=32, Hkv=8, D=128, page=64, max_pages=4, P=4, max_len=100, n=0, scale=1.0, o16=FAKE,
             o32=None, lse=FAKE, ws=None, wsb=0)
    a.update(kw)
    return ops.lib().ws_gqa_prompt(*a.values(), None)


@pytest.mark.parametrize("kw, rc, says", [
    (dict(cu=None), -1, "null"), (dict(o16=None), -1, "null"), (dict(ks=FAKE), -1, "null"),
    (dict(Hq=33), -1, "bad sizes"), (dict(B=2049), -1, "bad sizes"), (dict(n=65), -1, "bad sizes"),
    (dict(N=-1), -1, "bad sizes"), (dict(D=80), -1, "head_dim"), (dict(page=16), -1, "paging"),
    (dict(max_len=257), -1, "paging"), (dict(P=1 << 24), -1, "32-bit"), (dict(q=ODD), -1, "aligned"),
    (dict(scale=float("nan")), -1, "finite"), (dict(scale=float("inf")), -1, "finite"),
    (dict(N=1 << 30), -1, "exceed"), (dict(n=2), -3, "workspace"),
    (dict(n=2, ws=ctypes.c_void_p(0x1010), wsb=1 << 40), -1, "256-byte")])
def test_prompt_refusals(kw, rc, says):
    assert prompt(**kw) == rc and says in err()


def test_python_layer_wants_gpu_tensors():
    i = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises(ValueError, match="on a GPU"):
        ops.pages_extend(i, i[:, 0], i[:, 0], i[0], i[0, :1], 64, 4, 3)
    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="on a GPU"):
        ops.rope(x, x, i[0], torch.zeros(32))
    with pytest.raises(TypeError, match="tensor"):
        ops.gqa_prompt(x, None, None, i, i[0], i[0], 1.0, 3)
    with pytest.raises(ValueError, match="on a GPU"):
        ops.gqa8_decode_full(x, x, x, x, x, i, i[0], 1.0, 3)


def test_plans():
    pad = lambda n: -(-n // 256) * 256
    n, wsb = ops.gqa8_plan(16, 8, 96, 32768, 100)  # fp32 pieces
    assert n == 100 and wsb == pad((100 + 16) * 8 * 4) + (100 + 16) * 8 * 96 * 4
    n, _ = ops.gqa8_plan(4, 8, 128, 64, 0)  # at least two blocks a split
    assert n == 4
    with pytest.raises(ops.WsError, match="head_dim"):
        ops.gqa8_plan(4, 8, 80, 64)
    # 40 tokens of 8 sequences, 4 heads a KV head: at most 5 + 8 tiles of 32 rows a KV head,
    # or 2 + 8 of 128
    for fp8, tiles, rows in ((False, 13, 32), (True, 10, 128)):
        n, wsb = ops.gqa_prompt_plan(40, 8, 32, 8, 128, 32000, 4, fp8)
        assert n == tiles * 8 * 4 and wsb == pad(n * rows * 4) + n * rows * 128 * 4
    # long prompts fill the chip by their rows; one split needs no workspace
    assert ops.gqa_prompt_plan(8192, 1, 32, 8, 128, 8192) == (0, 0)
    assert ops.gqa_prompt_plan(40, 8, 32, 8, 128, 32000, 1) == (0, 0)
    # one token over a long cache is split, a short cache is not
    assert ops.gqa_prompt_plan(1, 1, 32, 8, 128, 100000)[0] > 8
    assert ops.gqa_prompt_plan(1, 1, 32, 8, 128, 100) == (0, 0)
    with pytest.raises(ops.WsError, match="bad sizes"):
        ops.gqa_prompt_plan(1, 1, 32, 5, 128, 100)


def test_rope_sections():
    assert ops.rope_sections([2, 1, 3]) == [0, 0, 1, 2, 2, 2]
    assert ops.rope_sections([3, 1, 2], interleaved=True) == [0, 1, 2, 0, 2, 0]
    assert ops.rope_sections([4]) == [0] * 4 and ops.rope_sections([0, 2]) == [1, 1]
    with pytest.raises(ValueError):
        ops._axis_bytes((0, 4))
    with pytest.raises(ValueError):
        ops._axis_bytes((0, 0.5))


def test_oracle_gives_every_page_once():
    """Growing sequences to the pool's end: no page twice, none lost."""
    rng = np.random.default_rng(0)
    P, page, B = 40, 32, 5
    table, lens = np.full((B, 16), -1, np.int32), np.zeros(B, np.int32)
    stack, free = rng.permutation(P).astype(np.int32), P
    for _ in range(40):
        n = rng.integers(0, 70, B)
        t2, l2, _, _, slots, f2 = R.extend(table, lens, n, stack, free, page, P, int(n.sum()))
        held = [int(x) for b in range(B) if l2[b] >= 0 for x in t2[b, :-(-int(l2[b]) // page)]]
        assert len(set(held)) == len(held)
        if (l2 < 0).any():
            break
        assert len(held) == P - f2 and set(held).isdisjoint(stack[:f2].tolist())
        assert (slots >= 0).all() and len(set(slots.tolist())) == len(slots)
        table, lens, free = t2, l2, f2
    assert free < 12


def test_quantise_rule():
    x = torch.tensor([[448.0, 1.0], [449.0, -1.0], [0.0, 0.0], [2.0 ** -130, 0.0], [1e38, 3e38]])
    q, s = R.quantise(x)
    assert s.view(torch.uint8).tolist() == [127, 128, 127, 1, 247]
    assert q.float()[0].tolist() == [448.0, 1.0] and q.float()[1].tolist() == [224.0, -0.5]


def decode16(**kw):
    a = dict(q=FAKE, kp=FAKE, vp=FAKE, table=FAKE, lens=FAKE, B=1, Hq=32, Hkv=8, D=128, page=64, max_pages=4,
             P=4, max_len=100, n=0, scale=1.0, out=FAKE, lse=FAKE, ws=None, wsb=0)
    a.update(kw)
    return ops.lib().ws_gqa_decode_partial(*a.values(), None)


LONG = dict(page=64, max_pages=1 << 19, P=600, n=16)


@pytest.mark.parametrize("call", (decode8, decode16))
@pytest.mark.parametrize("kw, fits", [
    # a batch of worst cases far above what any cache holds: the lengths decide, not max_len
    (dict(B=256, max_len=8192), True), (dict(B=2048, max_len=1 << 17), True),
    (dict(B=256, Hkv=1, Hq=4, max_len=1 << 23), True), (dict(B=1, Hkv=1, Hq=4, max_len=1 << 25), True),
    (dict(B=2048, max_len=1 << 22), False), (dict(B=2, Hkv=1, Hq=4, max_len=1 << 24), False),
    (dict(B=257, Hkv=1, Hq=4, max_len=1 << 24), True), (dict(B=2048, Hkv=16384, Hq=16384, max_len=64, P=1), False)])
def test_decode_block_range(call, kw, fits):
    """Refused only where 32-bit block numbers do not hold (what fits goes on to the
    workspace, which is missing)."""
    rc = call(**{**LONG, **kw})
    assert (rc == -3 and "workspace" in err()) if fits else (rc == -1 and "block index range" in err())


def test_plan_numbers_hold_to_the_limit():
    """The split plan's arithmetic (start of split g: floor(g T / n) from 32-bit products;
    split of a block: a quotient in 64-bit floating point) up to the largest total."""
    rng = np.random.default_rng(1)
    totals = [1, 31, 4096, 4097, (1 << 19) + 1, (1 << 31) - (1 << 16) - 1] + \
        [int(x) for x in np.exp2(rng.uniform(12, 31, 40)) if x < (1 << 31) - (1 << 16)]
    for T in totals:
        for grid in (1, 7, 512, 2048, 4095, 4096):
            n = min(grid, T)
            q, r = T // n, T - T // n * n
            g = np.arange(n + 1, dtype=np.int64)
            assert (g * r < 1 << 32).all()
            start = g * q + (g * r) // n
            assert (start == np.array([int(i) * T // n for i in g])).all() and start[-1] == T < 1 << 31
            for blk in (start[:-1], start[1:] - 1):  # a range's first and last block
                owner = np.ceil((blk + 1).astype(np.float64) * float(n) / float(T)).astype(np.int64) - 1
                assert (owner == g[:-1]).all()


@pytest.mark.parametrize("B, Hkv, D, fp8", [(1000, 8, 128, True), (2048, 8, 128, True), (256, 8, 64, False),
                                            (2000, 1, 128, True)])
def test_prompt_workspace_of_many_sequences(B, Hkv, D, fp8):
    """A batch of single tokens: pieces for the tiles that can be split (at most as many as
    shares), not for one of every sequence and KV head."""
    n, wsb = ops.gqa_prompt_plan(B, B, 4 * Hkv, Hkv, D, 8192, fp8=fp8)
    fill = 256 * 8  # the most workgroups at once, on 256 CUs
    assert n <= 2 * fill + 64 and n < B * Hkv + fill
    rows = 128 if fp8 else 32
    assert wsb <= n * rows * (D + 1) * 4 + 256 and wsb < 64 << 20


@pytest.mark.parametrize("kw, rc, says", [
    (dict(o16=None), -1, "out_bf16 is null"), (dict(o16=ODD), -1, "aligned"), (dict(q=None), -1, "null"),
    (dict(out=None), -1, "null"), (dict(Hq=33), -1, "heads"), (dict(D=40), -1, "head_dim"), (dict(n=16), -3, "workspace")])
def test_decode_full_refusals(kw, rc, says):
    a = dict(q=FAKE, kp=FAKE, vp=FAKE, table=FAKE, lens=FAKE, B=1, Hq=32, Hkv=8, D=128, page=64, max_pages=4,
             P=4, max_len=100, n=0, scale=1.0, o16=FAKE, out=FAKE, lse=FAKE, ws=None, wsb=0)
    a.update(kw)
    assert ops.lib().ws_gqa_decode_full(*a.values(), None) == rc and says in err()
