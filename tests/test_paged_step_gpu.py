"""Paged-cache operators as they are used together, and at the sizes where a
form, a list or an address changes.

Bound of the attention at sizes too large for the weights' distance from the
output, sum_j w_j |v_j - o|: |v_j - o| <= |v_j| + |o|, so that a rounding of
each weight by at most 2^-8 moves the output by at most
2^-8 (sum_j w_j |v_j| + |o|).
"""
import numpy as np
import pytest
import torch

from tests import helpers as H
from tests import paged_oracle as PO
from tests.test_paged_gpu import Step, check_plan, host, ints
from toyinfer_amd import attn

pytestmark = pytest.mark.gpu


def wide_attention(q, k, v, window, sinks):
    """o and sum_j w_j |v_j| in float64, a head at a time, where q lies."""
    n, hq, d = q.shape
    length, hkv = k.shape[:2]
    seen = torch.from_numpy(PO.visible(n, length, window, sinks)).to(q.device)
    o, size = torch.empty(n, hq, d, dtype=torch.float64, device=q.device), None
    size = torch.empty_like(o)
    for h in range(hq):
        g = h // (hq // hkv)
        s = q[:, h].double() @ k[:, g].double().t().contiguous() / d ** 0.5
        w = torch.softmax(torch.where(seen, s, -float("inf")), -1)
        vh = v[:, g].double()
        o[:, h], size[:, h] = w @ vh, w @ vh.abs()
    return o, size


def check_rows(got, q, k, v, window, sinks, what):
    o, size = wide_attention(q, k, v, window, sinks)
    bound = 2.0 ** -8 * (size + 2 * o.abs()) * (1 + 2.0 ** -6) + 2.0 ** -12 * size
    bad = ~((got.double() - o).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist())


class Wide(Step):
    def check(self, got=None):
        got = self.o if got is None else got
        assert (got[self.total:] == 3.0).all(), "rows behind the last request were written"
        for b in range(self.batch):
            rows = slice(int(self.start[b]), int(self.start[b + 1]))
            if rows.start < rows.stop:
                k, v = (x.to(self.dev) for x in self.kv[b])
                check_rows(got[rows], self.q_d[rows], k, v, self.window, self.sinks, b)


def shape_of(st):
    """(largest unit, split into pieces, more lists than lanes) of a made plan."""
    raw = st.plan.cpu().numpy()
    head = raw[:256].view(np.uint32)
    n, ranges = int(head[10]), int(head[12])
    every = raw[256:256 + 48 * (ranges + n)].view(np.uint32).reshape(-1, 12)
    rows = max(int(i[3]) for i in every[:ranges])
    return (next(r for r in (32, 64, 128, 256) if rows <= r), int(head[11]) > 0,
            ranges > max(1, 256 // st.hkv))


# Steps for the forms of the attention and the kinds of list.
FORMS = [
    (32, 8, 128, [(8192, 1)] * 3 + [(5000, 1)]),
    (32, 8, 128, [(300 + 9 * i, 1) for i in range(40)]),
    (32, 8, 128, [(512, 512)]),
    (32, 8, 128, [(4096, 16)]),
    (32, 8, 128, [(2048, 2048)]),
    (8, 8, 128, [(6000, 1000), (700, 64)]),
    (32, 8, 64, [(1024, 256)] * 8),
    (16, 8, 128, [(1371, 1371), (900, 1), (64, 5)]),
    (8, 8, 64, [(18000, 1)] * 16),
]


@pytest.mark.parametrize("case", range(len(FORMS)))
def test_each_form(dev, case):
    hq, hkv, d, requests = FORMS[case]
    st = Wide(dev, requests, hq, hkv, d, 16, seed=case)
    st.make_plan()
    H.sync()
    print(f"[paged] {hq}/{hkv} D={d} {requests[:3]}: {shape_of(st)}", flush=True)
    st.run()


def test_forms_are_reached(dev):
    """The steps above take units of every size, whole and in pieces, from lists
    of the lanes' own and drawn ones: a form that no step reaches any more is
    noticed."""
    shapes = set()
    for hq, hkv, d, requests in FORMS:
        st = Wide(dev, requests, hq, hkv, d, 16)
        st.make_plan()
        H.sync()
        check_plan(st)
        shapes.add(shape_of(st))
    assert {rows for rows, _, _ in shapes} == {32, 64, 128, 256}
    assert {pieces for _, pieces, _ in shapes} == {drawn for _, _, drawn in shapes} == {False, True}


@pytest.mark.parametrize("hq,hkv,d,requests", [
    (64, 1, 128, [(700, 3), (90, 90)]),        # one KV head, a group of 64
    (71, 1, 64, [(500, 2), (40, 40)]),         # rows of a token across units
    (9, 3, 128, [(3000, 1), (260, 130)]),      # 85 lanes per head, one workgroup of 256 left out
    (260, 260, 64, [(200, 1), (70, 20)]),      # more heads than compute units
])
def test_head_layouts(dev, hq, hkv, d, requests):
    print(f"[paged] heads {hq}/{hkv} D={d}", flush=True)
    Wide(dev, requests, hq, hkv, d, 16, seed=hq).run()


@pytest.mark.parametrize("hq,hkv,d,requests", [
    (25, 5, 128, [(2042, 373)]),                              # a last unit of 73 rows
    *[(8, 8, 128, [(6000, n)]) for n in (70, 96, 129, 160, 170, 200, 224)],
    (8, 8, 64, [(5000, 140), (3000, 200), (4000, 90)]),
    (16, 8, 128, [(7000, 300), (100, 1), (3000, 70)]),
])
def test_pieces_of_units_with_idle_waves(dev, hq, hkv, d, requests):
    """A split unit of fewer rows than its form's waves hold: the idle waves
    leave the next piece's results alone."""
    print(f"[paged] idle waves {hq}/{hkv} D={d} {requests}", flush=True)
    Wide(dev, requests, hq, hkv, d, 16, seed=hq).run()


@pytest.mark.parametrize("window,sinks", [(0, 0), (9000, 100)])
@pytest.mark.parametrize("ps", [8, 64])
def test_long_contexts(dev, ps, window, sinks):
    """Tables of several LDS fills: a fill holds 4096 keys at page size 8."""
    print(f"[paged] long, page size {ps} window {window}", flush=True)
    Wide(dev, [(40001, 1), (20000, 100), (33000, 9)], 8, 2, 128, ps, window, sinks, seed=ps).run()


def test_many_requests(dev):
    """A thousand decoded tokens: lists drawn by ticket, also of other heads."""
    rng = np.random.default_rng(4)
    Wide(dev, [(int(x), 1) for x in rng.integers(1, 700, 1000)], 16, 4, 128, 16, seed=4).run()


def test_pages_past_4_gib(dev):
    """Byte and element offsets beyond 32 bits, in the prologue's slots and in
    the attention's pages."""
    hq, hkv, d, ps = 8, 4, 128, 64
    page = ps * hkv * d
    pages = (2 ** 32 + 2 ** 28) // page          # element offsets past 2^32
    kc = torch.empty(pages, ps, hkv, d, dtype=torch.bfloat16, device=dev)
    vc = torch.empty_like(kc)
    length, new = 300, 40
    table = [pages - 1, 3, pages - 7, pages // 2 + 1, pages - 3]
    g = torch.Generator().manual_seed(1)
    def bf(*shape):
        return torch.randn(shape, generator=g).to(torch.bfloat16).to(dev)
    q, k, v = bf(length, hq, d), bf(length, hkv, d), bf(length, hkv, d)
    one = torch.ones(d, dtype=torch.bfloat16, device=dev)
    rope = torch.zeros(length, d // 2, 2, device=dev)
    rope[..., 0] = 1.0
    slots = [table[j // ps] * ps + j % ps for j in range(length)]
    q_out = torch.empty_like(q)
    print("[paged] prologue past 4 GiB", flush=True)
    attn.paged_qkv_prologue_bf16(q, k, v, one, one, rope, length, ints(range(length), dev),
                                 ints(slots, dev), length, 1e-6, q_out, kc, vc, pages, ps, page, hq,
                                 hkv, d)
    H.sync()
    rows_k = torch.stack([kc[s // ps, s % ps] for s in slots])
    rows_v = torch.stack([vc[s // ps, s % ps] for s in slots])
    assert torch.equal(rows_v, v)
    cs = np.stack([np.ones((length, d // 2)), np.zeros((length, d // 2))], -1)
    exp = PO.rms_rope(k.double().cpu().numpy(), np.ones(d), cs, 1e-6)
    assert (np.abs(rows_k.double().cpu().numpy() - exp) <= 2.0 ** -8 * np.abs(exp) * 1.02).all()
    qn = q_out[length - new:].contiguous()
    o = torch.empty_like(qn)
    plan = attn.paged_attention_plan_buffer(1, new, hq, hkv, d, dev)
    ws = attn.paged_attention_workspace(hq, hkv, d, dev)
    print("[paged] attention past 4 GiB", flush=True)
    attn.paged_attention_plan(ints([0, new], dev), ints([length], dev), 1, new, ps, 5, 0, 0, hq,
                              hkv, d, plan)
    attn.paged_attention_bf16(qn, kc, vc, o, ints(table, dev), plan, 1, new, pages, ps, page, 5, 0,
                              0, hq, hkv, d, ws)
    H.sync()
    check_rows(o, qn, rows_k, rows_v, 0, 0, "past 4 GiB")


def test_workspace_stays_zeroed(dev):
    """The counters that a call needs at zero are so after every call, also one
    that met infinities in hidden keys."""
    st = Step(dev, [(900, 1), (400, 120), (3000, 1)], 8, 2, 128, 16, seed=6)
    head = 4 * (st.hkv + 2)
    st.run()
    assert not st.ws[:head].any()
    st.v[int(st.table[1, 24]), 3] = float("inf")  # key 387 of the second request
    st.make_plan()
    for _ in range(3):
        st.attend()
    H.sync()
    assert not st.ws[:head].any()
    got = st.o.cpu().double()
    o, away, size = st.expect(1)
    first = int(st.start[1])
    rows = 387 - 280                               # tokens before it do not see it
    bound = 2.0 ** -8 * (away + o.abs()) * (1 + 2.0 ** -6) + 2.0 ** -12 * size
    assert ((got[first:first + rows] - o[:rows]).abs() <= bound[:rows]).all()
    assert not torch.isfinite(got[first + rows:first + 120]).any()


class Server:
    """A tiny serving loop over the four operators: requests with prompts of
    their own, taken in chunks, then decoded; random q, k, v per step."""

    def __init__(self, dev, prompts, hq, hkv, d, ps, window, sinks, rows, seed):
        self.dev, self.hq, self.hkv, self.d, self.ps = dev, hq, hkv, d, ps
        self.window, self.sinks, self.rows = window, sinks, rows
        self.batch, self.blocks, self.pages = len(prompts), 48, 160
        self.left = list(prompts)
        self.lens = [0] * self.batch
        g = torch.Generator().manual_seed(seed)
        self.g = g
        def bf(*shape, std=1.0):
            return (torch.randn(shape, generator=g) * std).to(torch.bfloat16).to(dev)
        self.bf = bf
        nan = float("nan")
        self.kc = torch.full((self.pages, ps, hkv, d), nan, dtype=torch.bfloat16, device=dev)
        self.vc = torch.full_like(self.kc, nan)
        self.qw, self.kw = bf(d), bf(d)
        ang = torch.rand(700, d // 2, generator=g) * 6.28
        self.rope = torch.stack([ang.cos(), ang.sin()], -1).float().to(dev)
        order = np.random.default_rng(seed).permutation(self.pages)
        self.free, self.free_d = order.tolist(), ints(order, dev)
        self.num_free = ints([self.pages], dev)
        self.table = ints(np.zeros((self.batch, self.blocks)), dev)
        self.ctx, self.new = ints([0] * self.batch, dev), ints([0] * self.batch, dev)
        self.query_start = ints([0] * (self.batch + 1), dev)
        self.seq_lens = ints([0] * self.batch, dev)
        self.positions, self.slots = ints([0] * rows, dev), ints([0] * rows, dev)
        self.status = ints([0, 0], dev)
        self.q, self.k, self.v = bf(rows, hq, d), bf(rows, hkv, d), bf(rows, hkv, d)
        self.q_out, self.o = torch.empty_like(self.q), torch.empty_like(self.q)
        self.plan = attn.paged_attention_plan_buffer(self.batch, rows, hq, hkv, d, dev)
        self.ws = attn.paged_attention_workspace(hq, hkv, d, dev)
        self.keys = [torch.zeros(0, hkv, d, dtype=torch.float64) for _ in prompts]
        self.vals = [torch.zeros(0, hkv, d, dtype=torch.bfloat16) for _ in prompts]

    def launch(self, stream=None):
        """The whole step: nothing of it depends on a length on the host."""
        attn.paged_tables_u32(self.ctx, self.new, self.batch, self.free_d, self.pages,
                              self.num_free, self.ps, self.table, self.blocks, self.rows,
                              self.query_start, self.seq_lens, self.positions, self.slots,
                              self.status, stream)
        attn.paged_attention_plan(self.query_start, self.seq_lens, self.batch, self.rows, self.ps,
                                  self.blocks, self.window, self.sinks, self.hq, self.hkv, self.d,
                                  self.plan, stream)
        attn.paged_qkv_prologue_bf16(self.q, self.k, self.v, self.qw, self.kw, self.rope, 700,
                                     self.positions, self.slots, self.rows, 1e-6, self.q_out,
                                     self.kc, self.vc, self.pages, self.ps,
                                     self.ps * self.hkv * self.d, self.hq, self.hkv, self.d, stream)
        attn.paged_attention_bf16(self.q_out, self.kc, self.vc, self.o, self.table, self.plan,
                                  self.batch, self.rows, self.pages, self.ps,
                                  self.ps * self.hkv * self.d, self.blocks, self.window, self.sinks,
                                  self.hq, self.hkv, self.d, self.ws, stream)

    def step(self, chunk, launch):
        """One step, with up to `chunk` prompt tokens per request, or one decoded
        token; checked against what the requests were given so far."""
        new = [min(chunk, x) if x else 1 for x in self.left]
        self.left = [x - n if x else 0 for x, n in zip(self.left, new)]
        self.ctx.copy_(ints(self.lens, self.dev))
        self.new.copy_(ints(new, self.dev))
        for t in (self.q, self.k, self.v):
            t.copy_(self.bf(*t.shape, std=1.2))
        self.o.fill_(3.0)
        H.sync()
        launch()
        H.sync()
        left, refused = host(self.status)
        assert refused == 0
        self.num_free.copy_(ints([left], self.dev))
        table, at = self.table.cpu().numpy().view(np.uint32), 0
        for b, n in enumerate(new):
            rows, before = slice(at, at + n), self.lens[b]
            self.lens[b] += n
            at += n
            cs = self.rope[before:before + n].double().cpu().numpy()
            k = PO.rms_rope(self.k[rows].double().cpu().numpy(), self.kw.double().cpu().numpy(), cs, 1e-6)
            self.keys[b] = torch.cat([self.keys[b], torch.from_numpy(k)])
            self.vals[b] = torch.cat([self.vals[b], self.v[rows].cpu()])
            length = self.lens[b]
            slot = [int(table[b, j // self.ps]) * self.ps + j % self.ps for j in range(length)]
            got_k = self.kc.view(-1, self.hkv, self.d)[slot]
            got_v = self.vc.view(-1, self.hkv, self.d)[slot]
            assert torch.equal(got_v.cpu(), self.vals[b]), b
            assert (got_k.cpu().double() - self.keys[b]).abs().max() <= 2.0 ** -8 * 8, b
            assert list(range(before, length)) == host(self.positions[rows]), b
            check_rows(self.o[rows], self.q_out[rows], got_k, got_v, self.window, self.sinks, b)
        assert (self.o[at:] == 3.0).all()
        used = {int(x) for b in range(self.batch) for x in table[b, :-(-self.lens[b] // self.ps)]}
        assert len(used) == sum(-(-x // self.ps) for x in self.lens) == self.pages - left


@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 4)])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (6, 2, 64)])
def test_serving_steps(dev, hq, hkv, d, window, sinks):
    """Chunked prompts and decoded tokens of several requests, the four
    operators one after the other on the current stream."""
    print(f"[paged] serving {hq}/{hkv} D={d} window {window}", flush=True)
    s = Server(dev, [130, 1, 300, 17, 64], hq, hkv, d, 16, window, sinks, 270, seed=hq + window)
    for _ in range(6):
        s.step(64, s.launch)


def test_serving_steps_captured(dev):
    """The same as one captured graph, replayed step after step with eager work
    between the replays."""
    s = Server(dev, [100, 33, 200], 16, 8, 128, 16, 0, 0, 140, seed=5)
    s.step(40, s.launch)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        s.launch(stream)
    other = Step(dev, [(700, 1), (90, 33)], 8, 2, 128, 16, seed=1)
    for _ in range(5):
        s.step(40, graph.replay)
        other.run()
    s.step(40, s.launch)


def test_paged_equals_contiguous(dev):
    """Decoding over pages against the contiguous decode attention over the same
    rows, and a prompt against the prefill attention: each is within the bound
    of the same exact result."""
    hq, hkv, d, b, length = 16, 8, 128, 3, 500
    st = Wide(dev, [(length, 1)] * b, hq, hkv, d, 16, seed=13, extra_rows=0)
    st.run()
    k = torch.stack([x[0] for x in st.kv]).to(dev)
    v = torch.stack([x[1] for x in st.kv]).to(dev)
    splits = attn.decode_default_splits(b, hq, hkv, d, length)
    o = torch.empty_like(st.o)
    attn.decode_attention_bf16(st.q_d, k, v, o, b, hq, hkv, d, None, length, length * hkv * d,
                               splits, attn.decode_workspace(b, hq, d, splits, dev))
    H.sync()
    for i in range(b):
        exact, size = wide_attention(st.q_d[i:i + 1], k[i], v[i], 0, 0)
        bound = 2 * (2.0 ** -8 * (size + 2 * exact.abs()) * 1.02 + 2.0 ** -12 * size)
        assert ((o[i:i + 1].double() - st.o[i:i + 1].double()).abs() <= bound).all()
    pt = Wide(dev, [(length, length)], hq, hkv, d, 16, seed=14, extra_rows=0)
    pt.run()
    o = torch.empty_like(pt.o)
    k, v = (x.to(dev) for x in pt.kv[0])
    attn.flash_attention_v1_bf16(pt.q_d, k, v, o, hq, hkv, d, length)
    H.sync()
    exact, size = wide_attention(pt.q_d, k, v, 0, 0)
    bound = 2 * (2.0 ** -8 * (size + 2 * exact.abs()) * 1.02 + 2.0 ** -12 * size)
    assert ((o.double() - pt.o.double()).abs() <= bound).all()


def test_binding_refuses_on_the_gpu(dev):
    """Tensors of another type, size, layout or device: refused, nothing
    written."""
    st = Step(dev, [(40, 1), (90, 3)], 8, 2, 128, 16)
    st.make_plan()
    H.sync()
    def attend(**kw):
        a = dict(q=st.q_d, k=st.k, v=st.v, o=st.o, table=st.table, plan=st.plan, ws=st.ws)
        a.update(kw)
        attn.paged_attention_bf16(a["q"], a["k"], a["v"], a["o"], a["table"], a["plan"], st.batch,
                                  st.rows, st.pages, st.ps, st.stride, st.blocks, 0, 0, st.hq,
                                  st.hkv, st.d, a["ws"])
    for kw in (dict(q=st.q_d.half()), dict(q=st.q_d[:-1]), dict(q=st.q_d.cpu()),
               dict(q=torch.cat([st.q_d, st.q_d], -1)[..., :st.d]), dict(k=st.k[1:]),
               dict(v=st.v.cpu()), dict(k=st.k.half()), dict(o=st.o.float()),
               dict(table=st.table.long()), dict(table=st.table[:1]), dict(plan=st.plan[:-256]),
               dict(plan=st.plan.cpu()), dict(ws=st.ws[:-16]), dict(ws=st.ws[16:]),
               dict(o=st.q_d), dict(ws=st.plan)):
        with pytest.raises(attn.ToyInferError):
            attend(**kw)
    H.sync()
    assert (st.o == 3.0).all()
    attend()
    H.sync()
    st.check()


def test_no_new_tokens(dev):
    """A step in which no request has a token: nothing is written."""
    st = Step(dev, [(40, 0), (0, 0), (300, 0)], 8, 2, 128, 16)
    st.run()
    assert (st.o == 3.0).all() and not st.ws[:4 * (st.hkv + 2)].any()


def test_graphs_that_share_a_workspace(dev):
    """Two captured steps with one workspace, replayed in turn on one stream with
    eager calls between, each with tickets, pieces and results of its own."""
    one = Step(dev, [(700, 1), (300, 40), (900, 1)], 8, 2, 128, 16, seed=21)
    two = Step(dev, [(3000, 1), (64, 64), (100, 5)], 8, 2, 128, 16, 70, 4, seed=22)
    two.ws = one.ws
    stream, graphs = torch.cuda.Stream(), []
    for st in (one, two):
        st.run()
        graph = torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            st.make_plan(stream)
            st.attend(stream)
        graphs.append(graph)
    for _ in range(3):
        for st, graph in zip((one, two), graphs):
            st.o.fill_(3.0)
            graph.replay()
        H.sync()
        one.check()
        two.check()
        one.attend()
        two.attend()
        H.sync()
        one.check()
        two.check()


def test_one_plan_on_two_streams(dev):
    """Two layers' calls with one plan at a time on two streams, each with a
    workspace of its own."""
    st = Step(dev, [(3000, 1), (500, 120), (60, 3)], 16, 8, 64, 16, seed=23)
    st.run()
    ws = attn.paged_attention_workspace(st.hq, st.hkv, st.d, dev)
    mine, other, first = st.o, torch.full_like(st.o, 3.0), st.o.clone()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    mine.fill_(3.0)
    H.sync()
    for _ in range(5):
        for stream, o, w in zip(streams, (mine, other), (st.ws, ws)):
            st.o, st.ws, keep = o, w, st.ws
            st.attend(stream)
            st.ws = keep
    H.sync()
    assert torch.equal(mine, first) and torch.equal(other, first)


class Early(Wide):
    """Requests with more new tokens than keys: rows before position 0 give 0,
    the others are as many tokens as keys."""

    def check(self, got=None):
        got = self.o if got is None else got
        assert (got[self.total:] == 3.0).all(), "rows behind the last request were written"
        for b, (length, new) in enumerate(self.requests):
            zero, first, end = int(self.start[b]), int(self.start[b]) + max(0, new - length), int(self.start[b + 1])
            assert (got[zero:first] == 0).all(), (b, "rows before position 0")
            if first < end:
                k, v = (x.to(self.dev) for x in self.kv[b])
                check_rows(got[first:end], self.q_d[first:end], k, v, self.window, self.sinks, b)


# With no window in forms of 32, 64, 128 (two) and 256 rows, the last in pieces.
EARLY = [
    (32, 8, 128, [(50, 100)]),
    (8, 8, 64, [(3005, 4096)]),
    (32, 8, 128, [(901, 1024)]),
    (64, 64, 64, [(30, 64), (71, 128), (1, 40), (9, 13)]),
    (32, 8, 128, [(53 - i, 100) for i in range(12)]),
    (8, 1, 128, [(9000, 1), (299, 2000), (5, 12)]),
]


@pytest.mark.parametrize("window,sinks", [(0, 0), (37, 2), (0x7FFFFFFE, 3), (0x7FFFFFFF, 0), (1 << 31, 5)])
@pytest.mark.parametrize("case", range(len(EARLY)))
def test_rows_on_both_sides_of_position_0(dev, case, window, sinks):
    """In each form, waves that hold rows before position 0 beside rows from it
    on, whatever window stands for none."""
    hq, hkv, d, requests = EARLY[case]
    st = Early(dev, requests, hq, hkv, d, 16, window, sinks, seed=case)
    st.make_plan()
    H.sync()
    print(f"[paged] before 0: {hq}/{hkv} D={d} {requests[:4]} window {window}: {shape_of(st)}", flush=True)
    st.run()
    if window == 0:
        assert shape_of(st)[0] == (32, 64, 128, 128, 256, 32)[case]


def test_head_counts_that_share_a_workspace(dev):
    """A call of few heads, whose units are in pieces, leaves the counters of a
    call of many heads alone."""
    few = Wide(dev, [(5000, 1), (3000, 40)], 16, 2, 128, 16, seed=31)
    many = Wide(dev, [(300, 1), (90, 40), (700, 3)], 130, 130, 64, 16, seed=32)
    ws = few.ws if few.ws.numel() > many.ws.numel() else many.ws
    few.ws = many.ws = ws
    for _ in range(2):
        few.run()
        assert shape_of(few)[1]
        assert not ws[:4 * (130 + 2)].any()
        many.o.fill_(3.0)
        many.run()
        assert shape_of(many)[2]
        few.o.fill_(3.0)


def put_nan(st, at):
    """NaN (or infinities) at (request, key, dim) of V, for every KV head."""
    for b, j, dim, x in at:
        st.v[int(st.table[b, j // st.ps]), j % st.ps, :, dim] = x


def check_nan(st, at):
    """An element is what its row's keys make of it: NaN or infinity by one that
    it sees, within the bound of the finite values' result elsewhere."""
    for b, (length, n) in enumerate(st.requests):
        rows = slice(int(st.start[b]), int(st.start[b + 1]))
        if not n:
            continue
        k, v = (x.to(st.dev) for x in st.kv[b])
        got, q = st.o[rows], st.q_d[rows]
        spoilt = torch.zeros(n, st.d, dtype=torch.bool, device=st.dev)
        seen = torch.from_numpy(PO.visible(n, length, st.window, st.sinks)).to(st.dev)
        for rb, j, dim, _ in at:
            if rb == b:
                spoilt[:, dim] |= seen[:, j]
        o, size = wide_attention(q, k, v, st.window, st.sinks)
        bound = 2.0 ** -8 * (size + 2 * o.abs()) * (1 + 2.0 ** -6) + 2.0 ** -12 * size
        ok = (got.double() - o).abs() <= bound
        spoilt = spoilt[:, None].expand_as(ok)
        assert ok[~spoilt].all(), (b, (~ok & ~spoilt).nonzero()[:3].tolist())
        assert not torch.isfinite(got[spoilt]).any(), b
    assert (st.o[st.total:] == 3.0).all() and not st.ws[:4 * (st.hkv + 2)].any()


NAN, INF = float("nan"), float("inf")
SPOILT = [
    (32, 8, 128, [(50, 50), (700, 3)], 0, 0, [(0, 33, 5, NAN), (1, 698, 9, INF)]),
    (8, 8, 64, [(3005, 3005)], 0, 0, [(0, 1000, 5, NAN), (0, 2900, 63, INF)]),
    (32, 8, 128, [(901, 901)], 0, 0, [(0, 0, 0, NAN), (0, 450, 127, NAN), (0, 900, 1, NAN)]),
    (32, 8, 128, [(100 + i, 100) for i in range(12)], 0, 0, [(b, 40 + 5 * b, b, NAN) for b in range(12)]),
    (8, 1, 128, [(9000, 1), (2000, 300), (15, 12)], 0, 0, [(1, 1800, 7, NAN), (2, 9, 7, -INF)]),
    (32, 8, 128, [(8192, 512)], 0, 0, [(0, 100, 3, NAN), (0, 8000, 77, NAN)]),
    (32, 8, 128, [(8192, 1), (5000, 4), (300, 1)], 1000, 4, [(0, 7191, 2, NAN), (1, 1, 2, NAN), (1, 3999, 3, INF)]),
    (6, 2, 64, [(5000, 300)], 1024, 16, [(0, 3700, 0, NAN), (0, 4800, 1, NAN)]),
]


@pytest.mark.parametrize("case", range(len(SPOILT)))
def test_values_that_are_not_finite(dev, case):
    """In each form, whole and in pieces: a value reaches the dims of the rows
    that see it, and no others."""
    hq, hkv, d, requests, window, sinks, at = SPOILT[case]
    st = Wide(dev, requests, hq, hkv, d, 16, window, sinks, seed=case)
    st.make_plan()
    H.sync()
    print(f"[paged] not finite: {hq}/{hkv} D={d} {requests[:3]}: {shape_of(st)}", flush=True)
    st.run()
    put_nan(st, at)
    for _ in range(2):
        st.o.fill_(3.0)
        st.attend()
        H.sync()
        check_nan(st, at)


@pytest.mark.parametrize("hq,d,requests", [
    (32, 64, [(5000, 5000), (900, 1)]),
    (64, 128, [(3300, 2300)]),
])
def test_more_spoilt_blocks_than_marks(dev, hq, d, requests):
    """NaN in one dim of every seventh token: more blocks of rows to compute again
    than a call keeps apart, some of them of units in pieces."""
    st = Wide(dev, requests, hq, hq, d, 16, seed=3)
    at = [(0, j, 11, NAN) for j in range(3, requests[0][0], 7)]
    put_nan(st, at)
    st.make_plan()
    st.attend()
    H.sync()
    print(f"[paged] more than the marks: {hq}/{hq} D={d}: {shape_of(st)}", flush=True)
    assert shape_of(st)[1]
    check_nan(st, at)


def time_of(f, n=20):
    f()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(n):
        f()
    end.record()
    H.sync()
    return start.elapsed_time(end) / n


@pytest.mark.parametrize("hq,hkv,d,requests,window,at", [
    (32, 8, 128, [(2048, 2048)], 0, (0, 5, 3, NAN)),        # seen by nearly all rows
    (32, 8, 128, [(2048, 2048)], 0, (0, 1500, 3, NAN)),
    (32, 8, 128, [(4000, 64)], 0, (0, 3980, 3, NAN)),       # in pieces
    (32, 8, 128, [(6000, 1)] * 8, 4096, (0, 1903, 3, NAN)),  # behind the window
])
def test_time_of_a_spoilt_call(dev, hq, hkv, d, requests, window, at):
    """One NaN does not turn a call into one of another order: only the blocks of
    rows that cannot tell it from a hidden one are computed again.  (All of a
    call's rows with NaN computed again took 300 to 4500 times the call.)"""
    st = Wide(dev, requests, hq, hkv, d, 16, window, seed=1)
    st.make_plan()
    clean = time_of(st.attend)
    put_nan(st, [at])
    spoilt = time_of(st.attend, 3)
    print(f"[paged] {requests[:2]} {1e3 * clean:.0f} us, with a NaN {1e3 * spoilt:.0f}", flush=True)
    assert spoilt < 30 * clean


def test_binding_refuses_caches_of_other_layouts(dev):
    """A transposed cache, or one whose pages lie elsewhere than the call says:
    refused by both calls that take one, nothing written."""
    st = Step(dev, [(40, 1), (90, 3)], 8, 2, 128, 16)
    st.make_plan()
    swapped = st.k.transpose(1, 2).contiguous()
    apart = torch.zeros(st.pages, 2, 16, 2, 128, dtype=torch.bfloat16, device=dev)[:, 0]
    rope = torch.zeros(99, 64, 2, device=dev)
    index = torch.zeros(st.rows, dtype=torch.int32, device=dev)
    new = st.q_d[:, :2].contiguous()
    w = torch.ones(128, dtype=torch.bfloat16, device=dev)
    for bad in (swapped, swapped.transpose(1, 2), apart):
        for k, v in ((bad, st.v), (st.k, bad)):
            with pytest.raises(attn.ToyInferError):
                attn.paged_attention_bf16(st.q_d, k, v, st.o, st.table, st.plan, st.batch, st.rows,
                                          st.pages, st.ps, st.stride, st.blocks, 0, 0, 8, 2, 128, st.ws)
            with pytest.raises(attn.ToyInferError):
                attn.paged_qkv_prologue_bf16(st.q_d, new, new, w, w, rope, 99, index, index, st.rows,
                                             1e-6, st.q_d, k, v, st.pages, st.ps, st.stride, 8, 2, 128)
    H.sync()
    assert (st.o == 3.0).all() and (apart == 0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (9000, 100)])
def test_long_contexts_miss_no_tile(dev, window, sinks, d):
    """Over tens of thousands of keys each weighs less than the elements' bound
    can see; the RMS over a request's elements sees a tile.  Its limit: a
    weight's rounding moves an element by at most 2^-8 w_j |v_j|, of random sign,
    which over the keys is 2^-8 of the output's own RMS, and the output's
    rounding is 2^-8 of it again: sqrt(2) 2^-8, below 2^-7.  64 of 33000 keys are
    4 % of it, which the same limit finds in an oracle that leaves them out."""
    st = Wide(dev, [(40001, 1), (20000, 33), (33000, 9)], 8, 2, d, 16, window, sinks, seed=d)
    st.run()
    rms = lambda x: x.square().mean().sqrt().item()
    for b, (length, n) in enumerate(st.requests):
        rows = slice(int(st.start[b]), int(st.start[b + 1]))
        k, v = (x.to(dev) for x in st.kv[b])
        o, _ = wide_attention(st.q_d[rows], k, v, window, sinks)
        error = rms(st.o[rows].double() - o) / rms(o)
        print(f"[paged] {length} keys, window {window}, D={d}: RMS {error:.5f}", flush=True)
        assert error < 2.0 ** -7, b
        gone = v.clone()
        first = length - length % 64 - 4 * 64
        gone[first:first + 64] = 0
        without, _ = wide_attention(st.q_d[rows], k, gone, window, sinks)
        assert rms(without - o) / rms(o) > 2.0 ** -7, b
