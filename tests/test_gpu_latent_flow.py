"""The latent path's operators together, as a program runs them: prompts, chunks and
single tokens of a ragged batch through MlaRequestPartition, tokens read back, sequences
that end and are replaced, the merge with a host share, other streams, captured steps."""
import numpy as np
import pytest
import torch

from scope_amd import ops
from scope_amd.cache import MlaRequestPartition
from tests import latent_oracle as L
from tests import request_oracle as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
C, PE, W = L.C, L.PE, L.W
INV = (1e4 ** (-torch.arange(PE // 2) / (PE // 2))).float()


class Model:
    """One layer's projections, made from the seed, and every sequence's exact latents."""

    def __init__(self, B, H):
        self.H, self.seed = H, 100
        self.weight = (1 + 0.2 * bf16_randn((C,), 3).float()).to(torch.bfloat16)
        self.lat = [torch.zeros((0, W), dtype=torch.float64) for _ in range(B)]

    def tokens(self, n_new):
        """(c, pe, q_nope, q_pe on the GPU, the first two as parts of one tensor; q_pe turned)."""
        N, self.seed = int(sum(n_new)), self.seed + 3
        kv, q = bf16_randn((N, W), self.seed, 2.0), bf16_randn((N, self.H, 192), self.seed + 1)
        qn = bf16_randn((N, self.H, C), self.seed + 2)
        pos = torch.from_numpy(np.concatenate(
            [np.arange(len(self.lat[b]), len(self.lat[b]) + n) for b, n in enumerate(n_new)]).astype(np.int32))
        x, _ = L.latents(kv[:, :C], kv[:, C:], pos, INV, True, 1.0, self.weight, 1e-6)
        at = 0
        for b, n in enumerate(n_new):
            self.lat[b] = torch.cat([self.lat[b], x[at:at + n]])
            at += n
        dkv, dq = kv.to(DEV), q.to(DEV)
        return dkv[:, :C], dkv[:, C:], qn.to(DEV), dq[..., 128:], R.rotate(q[..., 128:], pos, INV, None, True)

    def append(self, part, layer, c, pe, q_pe):
        return part.append(layer, c, pe, q_pe, INV.to(DEV), norm_weight=self.weight.to(DEV), adjacent=True)


def held(part, layer, b):
    """Sequence b's latents in the pages, in 64 bits."""
    sc = None if part.scale is None else part.scale[layer].cpu()
    return L.rows_of(part.latent[layer].cpu(), sc, part.page_table[b].cpu(), int(part.lens[b]), part.page_size,
                     part.scale_block)


def attention(q, n_new, kv, scale):
    N, H, _ = q.shape
    res = [torch.zeros((N, H, C), dtype=torch.float64), torch.zeros((N, H), dtype=torch.float64),
           torch.zeros((N, H, C), dtype=torch.float64), torch.zeros((N, H), dtype=torch.float64)]
    at = 0
    for b, n in enumerate(n_new):
        vis = [len(kv[b]) - n + i + 1 for i in range(n)]
        for r, x in zip(res, L.attend(q[at:at + n], kv[b], vis, scale, True)):
            r[at:at + n] = x
        at += n
    return res


@pytest.mark.parametrize("B, H, long", [(130, 16, 131008), (3, 48, 2000)])
def test_single_tokens_of_many_long_sequences(B, H, long):
    """Single tokens over bf16 pages with fp32 outputs, at and past the block index range of
    the decode kernel."""
    part = MlaRequestPartition(1, B, 1 << 17, 64, num_pages=long // 64 + 2 * B)
    part.latent.normal_(generator=torch.Generator(device=DEV).manual_seed(B))
    n = [3] * B
    n[1] = long
    part.begin(n)
    part.begin([1] * B)
    qn, qp = bf16_randn((B, H, C), 5), bf16_randn((B, H, PE), 6)
    out, lse = part.attend(0, qn.to(DEV), qp.to(DEV), 0.05)
    pool, table = part.latent[0].cpu(), part.page_table.cpu()
    for b in (0, 1, B - 1):
        kv = L.rows_of(pool, None, table[b], n[b] + 1, 64, 1)
        want_o, want_l, tol_o, tol_l = L.attend(torch.cat([qn, qp], -1).double()[b:b + 1], kv, [n[b] + 1], 0.05, True)
        R.check(out[b:b + 1], want_o, tol_o, f"out of {b}")
        R.check(lse[b:b + 1], want_l, tol_l, f"lse of {b}")


@pytest.mark.parametrize("bits, block, H", [(16, 1, 16), (8, 1, 16), (8, 32, 20), (16, 1, 5), (8, 8, 40)])
def test_requests_through_the_partition(bits, block, H):
    """Prompts, a chunk beside single tokens, single tokens, then a sequence that ends and
    another in its place.  The pages hold the exact latents to a rounding (with a scale for
    several tokens two: a raised scale rounds again), reading back gives what they hold, and
    the attention is that over it, with the turned q as it came out."""
    B, scale, ps = 3, 192 ** -0.5, 32
    m = Model(B, H)
    part = MlaRequestPartition(2, B, 256, ps, num_pages=14, bits=bits, scale_block=block)
    steps = [[70, 1, 40], [1, 60, 1], [1, 1, 1], [1, 1, 1], "release 0", [33, 1, 1], [1, 1, 1], [0, 2, 0]]
    for n_new in steps:
        if n_new == "release 0":
            part.release([0])
            m.lat[0] = m.lat[0][:0]
            continue
        c, pe, qn, q_pe, q_exact = m.tokens(n_new)
        part.begin(n_new)
        for layer in (1, 0):
            qr = m.append(part, layer, c, pe, q_pe)
            out, lse = part.attend(layer, qn, qr, scale)
        R.check(qr, q_exact, q_exact.abs() * 2.0 ** -8 + 1e-5, "q")
        kv = [held(part, 0, b) for b in range(B)]
        for b in range(B):
            want = m.lat[b]
            if len(want) == 0:
                continue
            step = want.abs() * (2.0 ** -8 if bits == 16 else 2.0 ** -4 * (2.125 if block > 1 else 1))
            # below e4m3's normal range, of a scale (at most its block's maximum / 224), twice
            top = float(want.abs().max()) if block > 1 else want.abs().amax(-1, keepdim=True)
            small = torch.as_tensor(0.0 if bits == 16 else top / 224 * 2.0 ** -10 * (2 if block > 1 else 1))
            R.check(kv[b], want, torch.maximum(step, step * 0 + small) + 1e-5, f"pages of {b}")
        start = [int(x) // 3 for x in part.lens]
        rows, rows_pe = part.read_back(0, start, [int(x) - s for x, s in zip(part.lens, start)])
        assert torch.equal(torch.cat([rows, rows_pe], 1).cpu().double(), torch.cat([k[s:] for k, s in zip(kv, start)]))
        q = torch.cat([qn, qr], -1).cpu().double()
        want_o, want_l, tol_o, tol_l = attention(q, n_new, kv, scale)
        R.check(out, want_o, tol_o, f"out {n_new}")
        R.check(lse, want_l, tol_l, f"lse {n_new}")
        o16, _ = part.attend(0, qn, qr, scale, out_dtype=torch.bfloat16)
        R.check(o16, want_o, tol_o + want_o.abs() * 2.0 ** -8, f"bf16 out {n_new}")
        assert part.len_dev.cpu().tolist() == part.lens.tolist() and int(part.free_dev) == part.free
    assert part.free == 14 - part._pages(part.lens)


def test_partition_refuses_before_anything_changes():
    part = MlaRequestPartition(1, 2, 128, 32, num_pages=5, bits=8, scale_block=16)
    q = lambda n, w=C: torch.zeros((n, 2, w), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="begin"):
        part.attend(0, q(2), q(2, PE), 1.0)
    part.begin([100, 0])
    for n, err in (([0, 40], MemoryError), ([29, 0], ValueError), ([0, -1], ValueError), ([1], ValueError)):
        with pytest.raises(err):
            part.begin(n)
    assert part.lens.tolist() == [100, 0] and part.free == 1 and int(part.free_dev) == 1
    for start, count in (([0, 0], [101, 0]), ([0, 1], [1, 0]), ([-1, 0], [1, 0]), ([0], [1]), ([0, 0], [-1, 0])):
        with pytest.raises(ValueError, match="start and count"):
            part.read_back(0, start, count)
    for bad in (q(99), q(101), q(100)[:, 0]):
        with pytest.raises(ValueError, match="100 tokens"):
            part.attend(0, bad, q(100, PE), 1.0)
    with pytest.raises(TypeError, match="out_dtype"):
        part.attend(0, q(100), q(100, PE), 1.0, torch.float16)
    part.begin([28, 32])
    assert part.free == 0 and part.len_dev.cpu().tolist() == [128, 32]
    for bad in (dict(page_size=48), dict(page_size=0), dict(bits=4), dict(scale_block=3), dict(scale_block=64),
                dict(scale_block=0)):
        with pytest.raises(ValueError):
            MlaRequestPartition(**{**dict(num_layers=1, batch=1, max_tokens=10, page_size=32, bits=8), **bad})


@pytest.mark.parametrize("bits", (16, 8))
def test_merge_with_a_host_share(bits):
    """The leading tokens of a prompt on the host, the rest in the pages: positions count
    both, queries that stand before the partition see nothing of it, and the two partials
    merge to attention over all tokens."""
    H, T, host, scale = 2, 90, 50, 0.1
    m = Model(1, H)
    c, pe, qn, q_pe, _ = m.tokens([T])
    part = MlaRequestPartition(1, 1, 64, 32, bits=bits)
    step = part.begin([T - host], pos_base=torch.tensor([host], dtype=torch.int32, device=DEV))
    assert step.positions.cpu().tolist() == list(range(host, T))
    m.append(part, 0, c[host:], pe[host:], q_pe[host:])
    every = torch.arange(T, dtype=torch.int32, device=DEV)
    rest = torch.empty((64, 64, W), dtype=torch.bfloat16, device=DEV)  # (a place for all T, for q's turn)
    qr = ops.latent_rope_append(c, pe, q_pe, every, INV.to(DEV), every, rest, norm_weight=m.weight.to(DEV), adjacent=True)
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    out, lse = ops.mla_prompt(qn, qr, part.latent[0], part.page_table, part.len_dev, cu, scale, 64,
                              latent_scale=part._scale(0), out_dtype=torch.float32)
    assert bool((out[:host] == 0).all()) and bool((lse[:host] == -np.inf).all())
    lat = torch.cat([rest.view(-1, W)[:host].cpu().double(), held(part, 0, 0)])
    q = torch.cat([qn, qr], -1).cpu().double()
    h_out, h_lse, _, _ = L.attend(q, lat[:host], [min(i + 1, host) for i in range(T)], scale, False)
    got, got_l = ops.lse_merge(out.view(-1, C), lse.view(-1), (h_out.float().view(-1, C).to(DEV), h_lse.float().view(-1).to(DEV)),
                               ops.PARTIAL_LSE_F32, out_dtype=torch.float32)
    o, l, to, tl = L.attend(q, lat, [i + 1 for i in range(T)], scale, True)
    R.check(got.view(T, H, C), o, to, "merged")
    R.check(got_l.view(T, H), l, tl + 1e-5, "merged lse")


def make_step(bits, B=5, H=16, ps=32, P=64, MP=8, N=5, n=1, block=1):
    """A forward step's buffers and its calls on them."""
    s = dict(table=torch.full((B, MP), -1, dtype=torch.int32, device=DEV),
             len=torch.zeros(B, dtype=torch.int32, device=DEV),
             n=torch.full((B,), n, dtype=torch.int32, device=DEV),
             stack=torch.randperm(P, generator=torch.Generator().manual_seed(1)).int().to(DEV),
             free=torch.tensor([P], dtype=torch.int32, device=DEV),
             x=torch.zeros((N, W), dtype=torch.bfloat16, device=DEV),
             q=torch.zeros((N, H, C + PE), dtype=torch.bfloat16, device=DEV),
             w=torch.ones(C, dtype=torch.bfloat16, device=DEV), inv=INV.to(DEV), sc=None)
    if bits == 16:
        s["pool"] = torch.zeros((P, ps, W), dtype=torch.bfloat16, device=DEV)
    else:
        s["pool"] = torch.zeros((P, ps, W), dtype=torch.uint8, device=DEV).view(R.E4M3)
        s["sc"] = torch.full((P, ps // block), 127, dtype=torch.uint8, device=DEV).view(R.E8M0)

    def run():
        st = ops.pages_extend(s["table"], s["len"], s["n"], s["stack"], s["free"], ps, P, N)
        qr = ops.latent_rope_append(s["x"][:, :C], s["x"][:, C:], s["q"][..., C:], st.positions, s["inv"], st.slots,
                                    s["pool"], s["sc"], s["w"])
        qn = s["q"][..., :C].contiguous()
        outs = []
        for splits in (0, 3):
            outs += ops.mla_prompt(qn, qr, s["pool"], s["table"], st.len_out, st.cu_new, 0.1, MP * ps, s["sc"], splits)
        if bits == 8 and n == 1:
            outs += ops.mla8_decode_full(qn, qr, s["pool"], s["sc"], s["table"], st.len_out, 0.1, MP * ps)
            outs += ops.mla8_decode_partial(qn, qr, s["pool"], s["sc"], s["table"], st.len_out, 0.1, MP * ps, 5)
        outs += ops.latent_gather(s["pool"], s["table"], st.cu_new, N, s["len"], s["sc"])
        s["len"].copy_(st.len_out)
        s["free"].copy_(st.free_out)
        return outs + [st.positions, st.slots, qr]

    return s, run


def state(s):
    return [s["table"], s["len"], s["free"], s["pool"].view(torch.uint8)] + \
        ([] if s["sc"] is None else [s["sc"].view(torch.uint8)])


@pytest.mark.parametrize("bits, n, block, H", [(8, 1, 1, 16), (16, 1, 1, 16), (8, 30, 32, 16), (16, 30, 1, 16),
                                               (8, 1, 8, 40), (8, 30, 1, 64)])
def test_captured_steps_replay(bits, n, block, H):
    """A step captured in a graph and replayed, with eager work between the replays: every
    replay is the eager step's, bit for bit."""
    make = lambda: make_step(bits, N=5 * n, n=n, block=block, H=H)
    se, eager = make()
    sg, run = make()
    run()  # (loads the library's kernels), then back to the start
    fresh, _ = make()
    for a, b in zip(state(sg), state(fresh)):
        a.copy_(b)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            outs = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(state(sg), state(fresh)):
        a.copy_(b)
    for i in range(6):
        for k in ("x", "q"):
            t = bf16_randn(tuple(se[k].shape), 50 + i).to(DEV)
            se[k].copy_(t)
            sg[k].copy_(t)
        want = eager()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), f"replay {i}"
        for a, b in zip(state(sg), state(se)):
            assert torch.equal(a, b), f"state after replay {i}"
        torch.zeros(1 << 20, device=DEV).add_(1.0)  # other work between the replays


@pytest.mark.parametrize("bits, n", [(8, 1), (16, 1), (8, 40)])
def test_two_graphs_and_streams_at_once(bits, n):
    """Two captured steps replayed on two streams at once, and the same calls on two streams
    eagerly: neither sees the other's workspaces.  (40 tokens of 64 heads: the latents are
    widened in a pass of their own.)"""
    make = lambda: make_step(bits, n=n, N=5 * n, P=80, MP=12, H=64 if n > 1 else 16)
    made, want_made = [make(), make()], [make(), make()]
    for i, ((s, _), (w, _)) in enumerate(zip(made, want_made)):
        for k in ("x", "q"):
            t = bf16_randn(tuple(s[k].shape), 7 + i).to(DEV)
            s[k].copy_(t)
            w[k].copy_(t)
    for (_, run) in made + want_made:
        run()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for (s, run) in made:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    torch.cuda.synchronize()
    for i in range(4):
        want = [run() for _, run in want_made]
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w)), f"replay {i}"
    want = [run() for _, run in want_made]
    torch.cuda.synchronize()
    got = []
    for (_, run), st in zip(made, streams):
        with torch.cuda.stream(st):
            got.append(run())
    torch.cuda.synchronize()
    for o, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w)), "eager on two streams"


@pytest.mark.parametrize("bits", (8, 16))
def test_single_tokens_beside_one_long_request(bits):
    """A token of each of 200 sequences, one of them long, and a step that holds a long prompt
    beside them."""
    B, H, ps, T = 200, 16, 64, 3000
    part = MlaRequestPartition(1, B, T + ps, ps, num_pages=B + T // ps + 2, bits=bits)
    m = Model(B, H)
    n_new = np.ones(B, np.int64)
    n_new[7] = T
    for n in (n_new, np.ones(B, np.int64)):
        N = int(n.sum())
        kv, qn = bf16_randn((N, W), 60 + N).to(DEV), bf16_randn((N, H, C), 61 + N).to(DEV)
        q_pe = bf16_randn((N, H, PE), 62 + N).to(DEV)
        step = part.begin(n)
        qr = m.append(part, 0, kv[:, :C], kv[:, C:], q_pe)
        out, lse = part.attend(0, qn, qr, 0.1)
        assert int(step.slots.min()) >= 0
        # the last token of every sequence, in 64 bits
        last = (step.cu_new[1:] - 1).cpu().long()
        q = torch.cat([qn, qr], -1)[last.to(DEV)].cpu().double()
        want = attention(q, [1] * B, [held(part, 0, b) for b in range(B)], 0.1)
        R.check(out[last.to(DEV)], want[0], want[2], "out")
        R.check(lse[last.to(DEV)], want[1], want[3], "lse")


def test_read_back_does_not_wait_for_the_device():
    part = MlaRequestPartition(1, 4, 256, 32, bits=8)
    part.latent.view(torch.uint8).zero_()
    part.scale.view(torch.uint8).fill_(127)
    part.begin([40, 3, 0, 70])
    part.read_back(0, [1, 0, 0, 5], [30, 3, 0, 60])  # (loads the library's kernels)
    x = torch.randn((8192, 8192), device=DEV, dtype=torch.bfloat16)
    y = x @ x
    end = torch.cuda.Event()
    torch.cuda.synchronize()
    for _ in range(300):  # some 250 ms, where the call below takes one
        torch.mm(x, x, out=y)
    end.record()
    c, pe = part.read_back(0, [1, 0, 0, 5], [30, 3, 0, 60])
    running = not end.query()
    torch.cuda.synchronize()
    assert running, "read_back() waited for the work ahead of it"
    assert c.shape == (93, C) and pe.shape == (93, PE) and not bool(c.any())


def test_partition_knows_its_device():
    part = MlaRequestPartition(1, 2, 128, 32, device="cuda")
    assert part.device == part.page_table.device and part.device.index is not None
    assert part.latent.device == part.device


@pytest.mark.parametrize("B, H, long, decodes", [
    (64, 128, 40000, True), (64, 128, 32 * 8191 - 2, True), (64, 128, 32 * 8191 - 1, False), (130, 16, 32 * 4032 - 1, False),
    (32, 32, 32 * 16000, True)])
def test_single_tokens_run_decode_as_far_as_it_goes(B, H, long, decodes, monkeypatch):
    """Single tokens over bf16 pages with fp32 outputs run the decode kernel up to the sizes it
    takes (a sequence of 128 heads counts once there), and the prompt kernel past them."""
    ran = []
    for name in ("mla_decode_partial", "mla_prompt"):
        real = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, _r=real, _n=name, **k: ran.append(_n) or _r(*a, **k))
    part = MlaRequestPartition(1, B, 1 << 19, 64, num_pages=long // 64 + 2 * B)
    part.latent.normal_(generator=torch.Generator(device=DEV).manual_seed(B))
    n = [3] * B
    n[1] = long
    part.begin(n)
    part.begin([1] * B)
    qn, qp = bf16_randn((B, H, C), 5), bf16_randn((B, H, PE), 6)
    out, lse = part.attend(0, qn.to(DEV), qp.to(DEV), 0.05)
    assert ran == ["mla_decode_partial" if decodes else "mla_prompt"]
    pool, table, heads = part.latent[0].cpu(), part.page_table.cpu(), [0, H // 2 + 1, H - 1]
    q = torch.cat([qn, qp], -1).double()[:, heads]
    for b in (0, 1, B - 1):
        kv = L.rows_of(pool, None, table[b], n[b] + 1, 64, 1)
        want_o, want_l, tol_o, tol_l = L.attend(q[b:b + 1], kv, [n[b] + 1], 0.05, True)
        R.check(out[b:b + 1, heads], want_o, tol_o, f"out of {b}")
        R.check(lse[b:b + 1, heads], want_l, tol_l, f"lse of {b}")
