"""The request-path operators together, as a program runs them: prompts, chunks and
single tokens of a ragged batch through GqaRequestPartition, sequences that end and
are replaced, the merge with a host share, other streams, and captured steps."""
import numpy as np
import pytest
import torch

from scope_amd import ops
from scope_amd.cache import GqaRequestPartition
from tests import request_oracle as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Model:
    """One layer's fused projections, made from the seed, and what every sequence's
    keys and values are (rotated in 64 bits)."""

    def __init__(self, B, Hq, Hkv, D, sections=None):
        self.Hq, self.Hkv, self.D = Hq, Hkv, D
        self.inv = (1e4 ** (-torch.arange(D // 2) / (D // 2))).float()
        self.axis = ops.rope_sections(sections) if sections else None
        self.axes = len(sections) if sections else 1
        self.k = [torch.zeros((0, Hkv, D), dtype=torch.float64) for _ in range(B)]
        self.v = [torch.zeros((0, Hkv, D), dtype=torch.float64) for _ in range(B)]
        self.seed = 100

    def tokens(self, n_new):
        """(q, k, v on the GPU as views of one tensor, q rotated, positions) of a step."""
        N, self.seed = int(sum(n_new)), self.seed + 1
        w = bf16_randn((N, (self.Hq + 2 * self.Hkv) * self.D), self.seed)
        cut = (self.Hq * self.D, self.Hkv * self.D, self.Hkv * self.D)
        q, k, v = (x.view(N, -1, self.D) for x in w.split(cut, 1))
        pos = np.concatenate([np.arange(len(self.k[b]), len(self.k[b]) + n) for b, n in enumerate(n_new)])
        pos = torch.from_numpy(np.stack([pos // (a + 1) for a in range(self.axes)]).astype(np.int32))
        kr = R.rotate(k, pos, self.inv, self.axis, False)
        at = 0
        for b, n in enumerate(n_new):
            self.k[b] = torch.cat([self.k[b], kr[at:at + n]])
            self.v[b] = torch.cat([self.v[b], v[at:at + n].double()])
            at += n
        dev = w.to(DEV)
        dq, dk, dv = (x.view(N, -1, self.D) for x in dev.split(cut, 1))
        return dq, dk, dv, R.rotate(q, pos, self.inv, self.axis, False), pos.to(DEV)

    def attention(self, q, n_new, scale, kv=None):
        """The step's (out, lse, bounds) over kv[b] = (k, v), the exact ones by default."""
        G = self.Hq // self.Hkv
        res = [torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64), torch.zeros_like(q),
               torch.zeros(q.shape[:2], dtype=torch.float64)]
        at = 0
        for b, n in enumerate(n_new):
            k, v = (self.k[b], self.v[b]) if kv is None else kv[b]
            vis = [len(k) - n + i + 1 for i in range(n)]
            for h in range(self.Hq):
                for r, x in zip(res, R.attend(q[at:at + n, h], k[:, h // G], v[:, h // G], vis, scale)):
                    r[at:at + n, h] = x
            at += n
        return res


def held(part, layer, b):
    """Sequence b's (k, v) in the pages, in 64 bits [n, Hkv, D]."""
    n, ps = int(part.lens[b]), part.page_size
    row = part.page_table[b].cpu()
    out = []
    for pool, sc in ((part.k, part.k_scale), (part.v, part.v_scale)):
        p = pool[layer].cpu()
        s = sc[layer].cpu() if sc is not None else None
        out.append(torch.stack([R.tokens_of(p, s, row, h, n, ps) for h in range(part.num_kv_heads)], 1))
    return out


@pytest.mark.parametrize("bits, D, sections", [(16, 64, None), (8, 64, None), (16, 128, [24, 20, 20]),
                                               (8, 96, [16, 16, 16])])
def test_requests_through_the_partition(bits, D, sections):
    """Prompts, a chunk beside single tokens, single tokens, then a sequence that
    ends and another in its place.  The pages hold the exact keys and values to a
    rounding, and the attention is that over what the pages hold: q is rounded to
    bf16 once after its rotation, which the oracle takes as it is."""
    B, Hq, Hkv, scale, ps = 3, 4, 2, D ** -0.5, 32
    m = Model(B, Hq, Hkv, D, sections)
    part = GqaRequestPartition(2, B, Hkv, D, 256, ps, num_pages=14, bits=bits)
    steps = [[70, 1, 40], [1, 60, 1], [1, 1, 1], [1, 1, 1], "release 0", [33, 1, 1], [1, 1, 1], [0, 2, 0]]
    for n_new in steps:
        if n_new == "release 0":
            part.release([0])
            m.k[0], m.v[0] = m.k[0][:0], m.v[0][:0]
            continue
        q, k, v, q_exact, pos = m.tokens(n_new)
        part.begin(n_new)
        for layer in (1, 0):
            qr = part.append(layer, q, k, v, m.inv.to(DEV), pos, pair_axis=m.axis)
            out, lse = part.attend(layer, qr, scale)
        R.check(qr, q_exact, q_exact.abs() * 2.0 ** -8 + 1e-5, "q")
        kv = []
        for b in range(B):
            kb, vb = held(part, 0, b)
            for got, want in ((kb, m.k[b]), (vb, m.v[b])):
                step = want.abs() * (2.0 ** -8 if bits == 16 else 2.0 ** -4)
                # below e4m3's normal range, of a row's scale (at most its maximum / 224)
                small = 0 if bits == 16 else want.abs().amax(-1, keepdim=True) / 224 * 2.0 ** -10
                R.check(got, want, torch.maximum(step, step * 0 + small) + 1e-5, f"pages of {b}")
            kv.append((kb, vb))
        want_o, want_l, tol_o, tol_l = m.attention(qr.cpu().double(), n_new, scale, kv)
        R.check(out, want_o, tol_o, f"out {n_new}")
        R.check(lse, want_l, tol_l, f"lse {n_new}")
        o16, _ = part.attend(0, qr, scale, out_dtype=torch.bfloat16)
        R.check(o16, want_o, tol_o + want_o.abs() * 2.0 ** -8, f"bf16 out {n_new}")
        assert part.len_dev.cpu().tolist() == part.lens.tolist() and int(part.free_dev) == part.free
    assert part.free == 14 - part._pages(part.lens)


def test_partition_refuses_before_anything_changes():
    part = GqaRequestPartition(1, 2, 1, 64, 128, 32, num_pages=5)
    with pytest.raises(RuntimeError, match="begin"):
        part.attend(0, torch.zeros((2, 1, 64), dtype=torch.bfloat16, device=DEV), 1.0)
    part.begin([100, 0])
    for n, err in (([0, 40], MemoryError), ([29, 0], ValueError), ([0, -1], ValueError), ([1], ValueError)):
        with pytest.raises(err):
            part.begin(n)
    assert part.lens.tolist() == [100, 0] and part.free == 1 and int(part.free_dev) == 1
    part.begin([28, 32])
    assert part.free == 0 and part.len_dev.cpu().tolist() == [128, 32]
    for bad in (dict(page_size=48), dict(head_dim=80), dict(bits=4)):
        with pytest.raises(ValueError):
            GqaRequestPartition(**{**dict(num_layers=1, batch=1, num_kv_heads=1, head_dim=64,
                                          max_tokens=10), **bad})


@pytest.mark.parametrize("bits", (16, 8))
def test_attend_refuses_what_is_not_the_step(bits):
    part = GqaRequestPartition(1, 2, 1, 64, 128, 32, bits=bits)
    part.begin([3, 2])
    q = torch.zeros((5, 1, 64), dtype=torch.bfloat16, device=DEV)
    for bad in (q[:4], torch.cat((q, q[:1])), q[:, 0]):
        with pytest.raises(ValueError, match="5 tokens"):
            part.attend(0, bad, 1.0)
    with pytest.raises(TypeError, match="out_dtype"):
        part.attend(0, q, 1.0, torch.float16)
    part.begin([1, 1])
    with pytest.raises(TypeError, match="out_dtype"):
        part.attend(0, q[:2], 1.0, torch.float16)


def test_merge_with_a_host_share():
    """The leading tokens of a prompt on the host, the rest in the pages: positions
    count both, queries that stand before the partition see nothing of it, and the
    two partials merge to attention over all tokens."""
    D, Hq, L, host = 64, 2, 90, 50
    m = Model(1, Hq, 1, D)
    q, k, v, _, pos = m.tokens([L])
    part = GqaRequestPartition(1, 1, 1, D, 64, 32)
    step = part.begin([L - host], pos_base=torch.tensor([host], dtype=torch.int32, device=DEV))
    assert torch.equal(step.positions, pos[0, host:])
    part.append(0, q[host:], k[host:], v[host:], m.inv.to(DEV))
    qr, kr = ops.rope(q, k, pos, m.inv.to(DEV))
    cu = torch.tensor([0, L], dtype=torch.int32, device=DEV)
    out, lse = ops.gqa_prompt(qr, part.k[0], part.v[0], part.page_table, part.len_dev, cu, 0.125, 64,
                              out_dtype=torch.float32)
    assert bool((out[:host] == 0).all()) and bool((lse[:host] == -np.inf).all())
    kc, vc, qc = kr.cpu().double()[:, 0], v.cpu().double()[:, 0], qr.cpu().double()
    h_out, h_lse = torch.zeros((L, Hq, D)), torch.zeros((L, Hq))
    for h in range(Hq):
        o, l, _, _ = R.attend(qc[:, h], kc[:host], vc[:host], [min(i + 1, host) for i in range(L)], 0.125)
        h_out[:, h], h_lse[:, h] = o.float(), l.float()
    got, got_l = ops.lse_merge(out, lse, (h_out.to(DEV), h_lse.to(DEV)), ops.PARTIAL_LSE_F32,
                               out_dtype=torch.float32)
    for h in range(Hq):
        o, l, to, tl = R.attend(qc[:, h], kc, vc, [i + 1 for i in range(L)], 0.125)
        R.check(got[:, h], o, to, "merged")
        R.check(got_l[:, h], l, tl + 1e-5, "merged lse")


def make_step(bits, B=5, Hq=8, Hkv=2, D=64, ps=32, P=64, MP=8, N=5, n=1):
    """A forward step's buffers and its calls on them."""
    s = dict(table=torch.full((B, MP), -1, dtype=torch.int32, device=DEV),
             len=torch.zeros(B, dtype=torch.int32, device=DEV),
             n=torch.full((B,), n, dtype=torch.int32, device=DEV),
             stack=torch.randperm(P, generator=torch.Generator().manual_seed(1)).int().to(DEV),
             free=torch.tensor([P], dtype=torch.int32, device=DEV),
             x=torch.zeros((N, (Hq + 2 * Hkv) * D), dtype=torch.bfloat16, device=DEV),
             inv=(1e4 ** (-torch.arange(D // 2) / (D // 2))).float().to(DEV))
    if bits == 16:
        s["pools"] = [torch.zeros((P, Hkv, ps, D), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        s["sc"] = [None, None]
    else:
        s["pools"] = [torch.zeros((P, Hkv, ps, D), dtype=torch.uint8, device=DEV).view(R.E4M3)
                      for _ in range(2)]
        s["sc"] = [torch.full((P, Hkv, ps), 127, dtype=torch.uint8, device=DEV).view(R.E8M0)
                   for _ in range(2)]

    def run():
        q, k, v = (t.view(N, -1, D) for t in s["x"].split((Hq * D, Hkv * D, Hkv * D), 1))
        st = ops.pages_extend(s["table"], s["len"], s["n"], s["stack"], s["free"], ps, P, N)
        qr = ops.rope_append(q, k, v, st.positions, s["inv"], st.slots, *s["pools"], *s["sc"])
        outs = list(ops.gqa_prompt(qr, *s["pools"], s["table"], st.len_out, st.cu_new, 0.125, MP * ps,
                                   *s["sc"]))
        outs += ops.gqa_prompt(qr, *s["pools"], s["table"], st.len_out, st.cu_new, 0.125, MP * ps,
                               *s["sc"], n_splits=3)
        if bits == 8 and n == 1:
            outs += ops.gqa8_decode_full(qr, *s["pools"], *s["sc"], s["table"], st.len_out, 0.125, MP * ps)
            outs += ops.gqa8_decode_partial(qr, *s["pools"], *s["sc"], s["table"], st.len_out, 0.125,
                                            MP * ps, 40)
        s["len"].copy_(st.len_out)
        s["free"].copy_(st.free_out)
        return outs + [st.positions, st.slots, qr]

    return s, run


def state(s):
    return [s["table"], s["len"], s["free"], *(t.view(torch.uint8) for t in s["pools"]),
            *(t.view(torch.uint8) for t in s["sc"] if t is not None)]


@pytest.mark.parametrize("bits, n", [(8, 1), (16, 1), (8, 30), (16, 30)])
def test_captured_steps_replay(bits, n):
    """A step captured in a graph and replayed, with eager work between the replays:
    every replay is the eager step's, bit for bit."""
    se, eager = make_step(bits, N=5 * n, n=n)
    sg, run = make_step(bits, N=5 * n, n=n)
    run()  # (loads the library's kernels), then back to the start
    fresh, _ = make_step(bits, N=5 * n, n=n)
    for a, b in zip(state(sg), state(fresh)):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            outs = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(state(sg), state(fresh)):
        a.copy_(b)
    for i in range(6):
        x = bf16_randn(tuple(se["x"].shape), 50 + i).to(DEV)
        se["x"].copy_(x)
        sg["x"].copy_(x)
        want = eager()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), f"replay {i}"
        for a, b in zip(state(sg), state(se)):
            assert torch.equal(a, b), f"state after replay {i}"
        torch.zeros(1 << 20, device=DEV).add_(1.0)  # other work between the replays


def test_two_graphs_and_streams_at_once():
    """Two captured steps replayed on two streams at once, and the same calls on two
    streams eagerly: neither sees the other's workspaces."""
    made = [make_step(8), make_step(8)]
    want_made = [make_step(8), make_step(8)]
    xs = [bf16_randn(tuple(made[0][0]["x"].shape), 7 + i).to(DEV) for i in range(2)]
    for (s, _), (w, _), x in zip(made, want_made, xs):
        s["x"].copy_(x)
        w["x"].copy_(x)
    made[0][1](), want_made[0][1](), made[1][1](), want_made[1][1]()
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
    """A token of each of 256 sequences, one of them long: the worst case of the batch (256
    times the longest) is past half a million blocks, and the step runs."""
    B, Hkv, G, D, ps, L = 256, 8, 1, 32, 64, 8200
    part = GqaRequestPartition(1, B, Hkv, D, L + ps, ps, num_pages=B + L // ps + 2, bits=bits)
    n_new = np.ones(B, np.int64)
    n_new[7] = L
    for n in (n_new, np.ones(B, np.int64)):
        step = part.begin(n)
        N = int(n.sum())
        w = bf16_randn((N, (G + 2) * Hkv * D), 60 + N).to(DEV)
        q, k, v = (x.view(N, -1, D) for x in w.split((G * Hkv * D, Hkv * D, Hkv * D), 1))
        inv = torch.zeros(D // 2, device=DEV)  # no turn: the keys are as they came, to a rounding
        qr = part.append(0, q, k, v, inv)
    assert int(step.slots.min()) >= 0
    out, lse = part.attend(0, qr, 0.2)
    want = [torch.zeros(t, dtype=torch.float64) for t in ((B, Hkv * G, D), (B, Hkv * G)) * 2]
    table, qc = part.page_table.cpu(), qr.cpu().double()
    pools = [(p[0].cpu(), None if s is None else s[0].cpu())
             for p, s in ((part.k, part.k_scale), (part.v, part.v_scale))]
    for b in range(B):
        for h in range(Hkv * G):
            n = int(part.lens[b])
            kb, vb = (R.tokens_of(p, s, table[b], h // G, n, ps) for p, s in pools)
            for r, x in zip(want, R.attend(qc[b:b + 1, h], kb, vb, [n], 0.2)):
                r[b, h] = x[0]
    want_o, want_l, tol_o, tol_l = want
    if bits == 16:
        tol_o = 2 * tol_o  # bf16 pieces: each off by another 2^-8 of its own weighted sum of |v|
    R.check(out, want_o, tol_o, "out")
    R.check(lse, want_l, tol_l, "lse")


def test_begin_and_release_do_not_wait_for_the_device():
    """Steps queued behind work that is still running: the calls return before it has
    ended, and every step gets its own counts."""
    B, ps, P = 4, 32, 60
    counts = [[5, 0, 40, 1], [1, 1, 1, 1], [33, 2, 0, 7], "release 2", [1, 64, 3, 1], [0, 1, 1, 90]]

    def run(part):
        steps = []
        for n in counts:
            if n == "release 2":
                part.release([2])
            else:
                steps.append((*part.begin(n), part.page_table.clone()))
        return steps

    make = lambda: GqaRequestPartition(1, B, 1, 32, 256, ps, num_pages=P)
    run(make())  # (loads the library's kernels)
    part = make()
    x = torch.randn((8192, 8192), device=DEV, dtype=torch.bfloat16)
    y = x @ x
    end = torch.cuda.Event()
    torch.cuda.synchronize()
    for _ in range(300):  # some 250 ms, where the calls below take one
        torch.mm(x, x, out=y)
    end.record()
    steps = run(part)
    running = not end.query()
    torch.cuda.synchronize()
    assert running, "begin() or release() waited for the work ahead of it"
    table, lens = np.full((B, 8), -1, np.int32), np.zeros(B, np.int32)
    stack, free, at = np.arange(P - 1, -1, -1).astype(np.int32), P, iter(steps)
    for n in counts:
        if n == "release 2":
            held = -(-int(lens[2]) // ps)
            stack[free:free + held] = table[2, :held]
            free, lens[2] = free + held, 0
            continue
        want = R.extend(table, lens, n, stack, free, ps, P, sum(n))
        len_out, cu, positions, slots, free_out, got_table = next(at)
        for got, w in zip((got_table, len_out, cu, positions, slots), want):
            assert got.cpu().tolist() == w.tolist(), n
        table, lens, free = want[0], want[1], want[5]
        assert int(free_out) == free


@pytest.mark.parametrize("bits", (16, 8))
def test_attend_single_tokens_round_the_decode_output(bits):
    """A step of one token of every sequence runs the same kernels for either output
    type: the bf16 output is the fp32 one, rounded, and the lse is the same."""
    B, Hq, Hkv, D = 3, 8, 2, 64
    part = GqaRequestPartition(1, B, Hkv, D, 2048, 64, bits=bits)
    for n in ([1500, 3, 70], [1, 1, 1]):
        part.begin(n)
        w = bf16_randn((sum(n), (Hq + 2 * Hkv) * D), 5 + n[0]).to(DEV)
        q, k, v = (x.view(sum(n), -1, D) for x in w.split((Hq * D, Hkv * D, Hkv * D), 1))
        qr = part.append(0, q, k, v, torch.ones(D // 2, device=DEV))
    want, want_l = part.attend(0, qr, 0.125)
    out, lse = part.attend(0, qr, 0.125, torch.bfloat16)
    assert out.dtype == torch.bfloat16 and torch.equal(out, want.bfloat16()) and torch.equal(lse, want_l)


def test_partition_knows_its_device():
    """A partition on "cuda" stays on the device that was current when it was made: its
    counts go there by number."""
    part = GqaRequestPartition(1, 2, 1, 64, 128, 32, device="cuda")
    assert part.device == part.page_table.device and part.device.index is not None
    assert part._to_device([1, 2], torch.int32).device == part.page_table.device


def test_decode_full_in_two_graphs_at_once():
    """Each captured call has a workspace of its own: two graphs replayed on two streams at
    once, with eager calls between the replays, give the eager results bit for bit."""
    B, Hkv, G, D, L = 2, 2, 4, 128, 3000  # (split rows: pieces in the workspace)
    made = []
    for i in range(2):
        k, v = (bf16_randn((B * 47, Hkv, 64, D), 70 + 2 * i + j).to(DEV) for j in range(2))
        table = torch.arange(B * 47, dtype=torch.int32, device=DEV).view(B, 47).flip(0).contiguous()
        lens = torch.tensor([L, L - 100 * i], dtype=torch.int32, device=DEV)
        made.append((bf16_randn((B, Hkv * G, D), 80 + i).to(DEV), k, v, table, lens, D ** -0.5, L))
    want = [ops.gqa_decode_full(*a) for a in made]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for a in made:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.gqa_decode_full(*a))
        graphs.append(g)
    for i in range(6):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w, a in zip(outs, want, made):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1]), f"replay {i}"
            assert torch.equal(ops.gqa_decode_full(*a)[0], w[0]), f"eager after replay {i}"
