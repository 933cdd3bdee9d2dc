"""Paged-cache operators on the GPU against plain 64-bit forms.

Attention's bound, from the kernels' roundings: each weight is rounded to bf16
once, the same value in numerator and denominator, so a weight's relative error
d <= 2^-8 moves the output by at most sum_j w_j d |v_j - o|; the output is
rounded once, 2^-8 |o|; scores (128 products summed in fp32, |q||k|/sqrt(D) of
about ten) and exponentials stay below 2^-12 of a weight, which moves it by at
most 2^-12 sum_j w_j |v_j|.  The factor 1 + 2^-6 holds the second-order terms.
"""
import numpy as np
import pytest
import torch

from tests import helpers as H
from tests import paged_oracle as PO
from toyinfer_amd import attn

pytestmark = pytest.mark.gpu


def ints(v, dev):
    return torch.from_numpy(np.asarray(v, np.uint32).view(np.int32).copy()).to(dev)


def host(t):
    return t.cpu().numpy().view(np.uint32).tolist()


# ------------------------------------------------------------------ tables

def run_tables(dev, context, new, free, ps, blocks, rows, capacity=None):
    rng = np.random.default_rng(5)
    table = rng.integers(0, 1000, (len(context), blocks)).astype(np.uint32)
    cap = len(free) if capacity is None else capacity
    out = {k: torch.full((n,), 77, dtype=torch.int32, device=dev) for k, n in
           (("query_start", len(context) + 1), ("seq_lens", len(context)), ("positions", rows),
            ("slots", rows), ("status", 2))}
    bt = ints(table, dev)
    attn.paged_tables_u32(ints(context, dev), ints(new, dev), len(context),
                          ints(list(free) + [999] * (cap - len(free)), dev), cap,
                          ints([len(free)], dev), ps, bt, blocks, rows, out["query_start"],
                          out["seq_lens"], out["positions"], out["slots"], out["status"])
    H.sync()
    exp = PO.tables(context, new, list(free), ps, table, rows)
    got = [host(out[k]) for k in ("query_start", "seq_lens", "positions", "slots")]
    for name, g, e in zip(("query_start", "seq_lens", "positions", "slots"), got, exp):
        assert g == [int(x) for x in e], name
    assert (bt.cpu().numpy().view(np.uint32) == exp[4]).all(), "block tables"
    assert host(out["status"]) == exp[5]


TABLES = {
    "one token": ([0], [1], 8, 4, 1),
    "page ends": ([7, 8, 9, 15, 16], [1, 1, 1, 1, 1], 8, 4, 5),
    "idle and empty": ([0, 5, 0, 40], [0, 0, 3, 0], 16, 4, 8),
    "prompts": ([0, 100, 3], [300, 29, 1], 16, 24, 400),
    "one long": ([17], [5000], 16, 400, 5017),
}


@pytest.mark.parametrize("name", TABLES)
def test_tables(dev, name):
    context, new, ps, blocks, rows = TABLES[name]
    run_tables(dev, context, new, range(500, 1100), ps, blocks, rows)


@pytest.mark.parametrize("batch", [1, 255, 256, 257, 1031, 4096])
def test_tables_batches(dev, batch):
    rng = np.random.default_rng(batch)
    context, new = rng.integers(0, 60, batch).tolist(), rng.integers(0, 5, batch).tolist()
    run_tables(dev, context, new, rng.permutation(9000).tolist(), 8, 9, sum(new) + 3)


def test_tables_refusals(dev):
    """Too few pages, a row past max_blocks, too few token rows: the request
    takes nothing, those after it keep what is left."""
    run_tables(dev, [0, 0, 8, 5], [16, 30, 8, 3], range(3), 8, 8, 64)     # the second starves
    run_tables(dev, [0, 60, 0], [9, 9, 9], range(20), 8, 8, 64)           # the second is too long
    run_tables(dev, [0, 0, 0], [9, 9, 9], range(20), 8, 8, 20)            # no rows for the third
    run_tables(dev, [3, 4], [2, 3], [], 8, 8, 8, capacity=2)              # none needed, none there
    run_tables(dev, [0xFFFFFFF0, 4], [0xFFFFFFFF, 3], range(5), 8, 8, 8)  # lengths of any content


def test_tables_num_free_over_capacity(dev):
    """*num_free past the array counts as the array's length."""
    bt = ints(np.zeros((1, 4)), dev)
    out = [ints([0] * 8, dev) for _ in range(5)]
    attn.paged_tables_u32(ints([0], dev), ints([8], dev), 1, ints([11, 12], dev), 2,
                          ints([4000000000], dev), 8, bt, 4, 8, *out)
    H.sync()
    assert host(bt[0, :1]) == [12] and host(out[4])[:2] == [1, 0]


# ---------------------------------------------------------------- prologue

@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (32, 8, 128), (5, 1, 64), (12, 2, 64),
                                      (1, 1, 128), (40, 40, 128)])
@pytest.mark.parametrize("t", [1, 7, 130])
def test_prologue(dev, hq, hkv, d, t):
    """Bound: the fp32 steps stay below 2^-16 of the two products' sizes, one
    rounding to bf16 (2^-8) follows.  Rows of slots not named keep their bytes,
    in caches that share one array, a page of K beside one of V."""
    ps, pages, positions = 16, 2 * t + 3, 97
    rng = np.random.default_rng(hq * t + d)
    def bf(*shape, std=1.0):
        return (torch.from_numpy(rng.standard_normal(shape) * std)).to(torch.bfloat16)
    q, k, v = bf(t, hq, d, std=3.0), bf(t, hkv, d, std=0.1), bf(t, hkv, d)
    qw, kw = bf(d), bf(d)
    rope = torch.from_numpy(rng.uniform(-1, 1, (positions, d // 2, 2))).float()
    pos = rng.integers(0, positions, t)
    slot = rng.permutation(pages * ps)[:t].astype(np.uint32)
    if t > 3:
        slot[1], slot[2], pos[3] = 0xFFFFFFFF, pages * ps, 5000  # no slot; past the caches; past the table
    both = bf(pages, 2, ps, hkv, d)
    dev_both = both.to(dev)
    k_cache, v_cache = dev_both[:, 0], dev_both[:, 1]
    q_out = torch.empty_like(q, device=dev)
    attn.paged_qkv_prologue_bf16(q.to(dev), k.to(dev), v.to(dev), qw.to(dev), kw.to(dev),
                                 rope.to(dev), positions, ints(pos, dev), ints(slot, dev), t, 1e-6,
                                 q_out, k_cache, v_cache, pages, ps, 2 * ps * hkv * d, hq, hkv, d)
    H.sync()
    cs = rope.double().numpy()[np.minimum(pos, positions - 1)]
    wide = np.abs(cs).sum(-1)
    live = slot < pages * ps
    for got, x, w in ((q_out.cpu(), q, qw), (k_cache.cpu().reshape(-1, hkv, d), k, kw)):
        x, w = x.double().numpy(), w.double().numpy()
        exp = PO.rms_rope(x, w, cs, 1e-6)
        y = np.abs(PO.rms_rope(x, w, np.stack([np.ones_like(wide), np.zeros_like(wide)], -1), 1e-6))
        half = d // 2
        terms = np.tile((y[..., :half] + y[..., half:]) * wide[:, None], 2)
        g = got.double().numpy()
        if g.shape != exp.shape:
            g, exp, terms = g[slot[live]], exp[live], terms[live]
        assert (np.abs(g - exp) <= 2.0 ** -8 * np.abs(exp) * 1.001 + 2.0 ** -16 * terms).all()
    want = both.clone()
    rows_k, rows_v = want[:, 0].clone().view(-1, hkv, d), want[:, 1].clone().view(-1, hkv, d)
    rows_v[slot[live].astype(np.int64)] = v[torch.from_numpy(live)]
    assert torch.equal(v_cache.cpu().reshape(-1, hkv, d), rows_v)
    untouched = np.setdiff1d(np.arange(pages * ps), slot[live])
    assert torch.equal(k_cache.cpu().reshape(-1, hkv, d)[untouched], rows_k[untouched])


def test_prologue_in_place(dev):
    """q_out may be q."""
    t, hq, hkv, d, ps = 9, 6, 2, 128, 8
    g = torch.Generator().manual_seed(3)
    def bf(*shape):
        return torch.randn(shape, generator=g).to(torch.bfloat16).to(dev)
    q, k, v, w = bf(t, hq, d), bf(t, hkv, d), bf(t, hkv, d), bf(d)
    rope, pos, slot = torch.rand(50, d // 2, 2, device=dev), ints(range(t), dev), ints(range(t), dev)
    res = []
    for out in (torch.empty_like(q), q):
        kc, vc = torch.zeros(2, ps, hkv, d, dtype=torch.bfloat16, device=dev), bf(2, ps, hkv, d)
        attn.paged_qkv_prologue_bf16(q, k, v, w, w, rope, 50, pos, slot, t, 1e-6, out, kc, vc, 2,
                                     ps, ps * hkv * d, hq, hkv, d)
        res.append((out.clone(), kc))
    H.sync()
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])


# --------------------------------------------------------------- attention

class Step:
    """A batch over caches whose unwritten rows and unused pages hold NaN."""

    def __init__(self, dev, requests, hq, hkv, d, ps, window=0, sinks=0, seed=0, std=1.5,
                 extra_rows=3, interleaved=False):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.dev, self.hq, self.hkv, self.d, self.ps = dev, hq, hkv, d, ps
        self.window, self.sinks, self.requests = window, sinks, requests
        self.batch = len(requests)
        lens = [length for length, _ in requests]
        self.blocks = max(1, max(-(-x // ps) for x in lens)) + 1
        need = [-(-x // ps) for x in lens]
        self.pages = sum(need) + 2
        order = rng.permutation(self.pages)
        table = np.full((self.batch, self.blocks), 0xFFFFFFFF, np.uint32)
        both = torch.full((self.pages, 2, ps, hkv, d), float("nan"), dtype=torch.bfloat16)
        self.kv, at = [], 0
        for b, x in enumerate(lens):
            k = torch.randn(x, hkv, d, generator=g).to(torch.bfloat16)
            v = torch.randn(x, hkv, d, generator=g).to(torch.bfloat16)
            self.kv.append((k, v))
            for j in range(need[b]):
                page = order[at + j]
                table[b, j] = page
                rows = min(ps, x - j * ps)
                both[page, 0, :rows] = k[j * ps:j * ps + rows]
                both[page, 1, :rows] = v[j * ps:j * ps + rows]
            at += need[b]
        if interleaved:
            self.both = both.to(dev)
            self.k, self.v, self.stride = self.both[:, 0], self.both[:, 1], 2 * ps * hkv * d
        else:
            self.k, self.v = both[:, 0].contiguous().to(dev), both[:, 1].contiguous().to(dev)
            self.stride = ps * hkv * d
        news = [n for _, n in requests]
        self.total = sum(news)
        self.rows = self.total + extra_rows
        self.start = np.concatenate([[0], np.cumsum(news)])
        self.q = (torch.randn(max(1, self.rows), hq, d, generator=g) * std).to(torch.bfloat16)
        self.q_d, self.table = self.q.to(dev), ints(table, dev)
        self.query_start, self.seq_lens = ints(self.start, dev), ints(lens, dev)
        self.o = torch.full((self.rows, hq, d), 3.0, dtype=torch.bfloat16, device=dev)
        self.plan = attn.paged_attention_plan_buffer(self.batch, self.rows, hq, hkv, d, dev)
        self.ws = attn.paged_attention_workspace(hq, hkv, d, dev)

    def make_plan(self, stream=None):
        attn.paged_attention_plan(self.query_start, self.seq_lens, self.batch, self.rows, self.ps,
                                  self.blocks, self.window, self.sinks, self.hq, self.hkv, self.d,
                                  self.plan, stream)

    def attend(self, stream=None):
        attn.paged_attention_bf16(self.q_d, self.k, self.v, self.o, self.table, self.plan,
                                  self.batch, self.rows, self.pages, self.ps, self.stride,
                                  self.blocks, self.window, self.sinks, self.hq, self.hkv, self.d,
                                  self.ws, stream)

    def expect(self, b):
        """Request b's rows: o, and the two sizes of PO.attention."""
        if not hasattr(self, "_exp"):
            self._exp = {}
        if b not in self._exp:
            k, v = self.kv[b]
            q = self.q[self.start[b]:self.start[b + 1]]
            self._exp[b] = PO.attention(q.double(), k.double(), v.double(), self.window, self.sinks)
        return self._exp[b]

    def check(self, got=None):
        got = (self.o if got is None else got).cpu().double()
        assert (got[self.total:] == 3.0).all(), "rows behind the last request were written"
        for b in range(self.batch):
            o, away, size = self.expect(b)
            g = got[self.start[b]:self.start[b + 1]]
            bound = 2.0 ** -8 * (away + o.abs()) * (1 + 2.0 ** -6) + 2.0 ** -12 * size
            bad = ~((g - o).abs() <= bound)
            assert not bad.any(), (f"request {b} {self.requests[b]}: {int(bad.sum())} of "
                                   f"{bad.numel()}, first at {bad.nonzero()[0].tolist()}: "
                                   f"{g[bad][0]} for {o[bad][0]}")

    def run(self):
        self.make_plan()
        H.sync()
        check_plan(self)
        self.attend()
        H.sync()
        self.check()


def check_plan(st):
    """The plan's lists as the attention kernels read them: every row of every
    request once, every tile of a unit once, partial blocks inside the
    workspace, before a kernel relies on it."""
    raw = st.plan.cpu().numpy()
    head = raw[:256].view(np.uint32)
    n, ranges = int(head[10]), int(head[12])
    lanes = max(1, 256 // st.hkv)
    assert lanes <= ranges
    every = raw[256:256 + 48 * (ranges + n)].view(np.uint32).reshape(-1, 12)
    items = []
    for i in every[:ranges]:
        while i[3]:
            items.append(i)
            if i[11] == 0xFFFFFFFF:
                break
            i = every[i[11]]
    assert len(items) == n
    group = st.hq // st.hkv
    units, blocks = {}, []
    for it in items:
        req, token0, row0, rows = (int(x) for x in it[:4])
        assert req < st.batch and 1 <= rows <= 256 and token0 == st.start[req]
        key_end, low, sink = int(it[5]), int(it[6]), int(it[7])
        assert key_end <= st.requests[req][0] and sink <= low
        units.setdefault((req, row0, rows, key_end, low, sink), []).append(it)
    seen = {}
    for (req, row0, rows, key_end, low, sink), its in units.items():
        tiles = (key_end - 1) // 64 + 1 - low + sink if key_end else 0
        spans = sorted((int(i[8]), int(i[9])) for i in its)
        assert spans[0][0] == 0 and spans[-1][1] == tiles
        assert all(a[1] == b[0] for a, b in zip(spans, spans[1:]))
        if len(its) > 1:
            nb = -(-rows // 32)
            for i in its:
                assert i[10] != 0xFFFFFFFF
                blocks += range(int(i[10]), int(i[10]) + nb)
        else:
            assert its[0][10] == 0xFFFFFFFF
        seen.setdefault(req, []).append((row0, row0 + rows))
    assert len(blocks) == len(set(blocks)) and max(blocks, default=0) < 16 * lanes
    for b, (_, new) in enumerate(st.requests):
        spans = sorted(seen.get(b, []))
        assert [s for s, _ in spans] == [0, *[e for _, e in spans[:-1]]][:len(spans)]
        assert (spans[-1][1] if spans else 0) == new * group


HEADS = [(16, 8, 128), (32, 8, 128), (32, 8, 64), (6, 2, 128), (5, 1, 64), (8, 8, 128)]
BATCHES = {
    "one token": [(1, 1)],
    "lengths around a tile": [(n, 1) for n in (1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200)],
    "idle requests": [(40, 0), (17, 1), (0, 0), (300, 2), (64, 0)],
    "prompt": [(150, 150)],
    "chunk": [(333, 70)],
    "mixed": [(90, 90), (500, 1), (77, 5), (260, 33), (1, 1), (700, 1)],
}


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("name", BATCHES)
def test_attention(dev, name, hq, hkv, d):
    print(f"[paged] {name} {hq}/{hkv} D={d}", flush=True)
    Step(dev, BATCHES[name], hq, hkv, d, 16, seed=hq + d).run()


@pytest.mark.parametrize("ps", [8, 16, 32, 64, 128, 512])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_page_sizes(dev, ps, d):
    print(f"[paged] page size {ps} D={d}", flush=True)
    Step(dev, [(700, 1), (130, 40), (515, 3)], 8, 2, d, ps, seed=ps, interleaved=ps in (8, 64)).run()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (64, 0), (100, 70), (300, 4),
                                          (0xFFFFFFFF, 5), (40, 0xFFFFFFFF), (1 << 31, 0)])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (6, 2, 64)])
def test_attention_window(dev, window, sinks, hq, hkv, d):
    print(f"[paged] window {window} sinks {sinks} {hq}/{hkv} D={d}", flush=True)
    Step(dev, [(600, 1), (130, 130), (420, 50), (9, 2), (333, 4)], hq, hkv, d, 16, window, sinks,
         seed=3).run()


@pytest.mark.parametrize("window,sinks", [(0, 0), (500, 4)])
@pytest.mark.parametrize("hq,hkv,d,requests", [
    (16, 8, 128, [(5000, 1)]),                      # split over the lanes, one token
    (32, 8, 128, [(3000, 40)]),                     # 160 rows
    (4, 1, 64, [(2100, 300)]),                      # few units, many lanes
    (1, 1, 128, [(4100, 1), (10, 1), (900, 64)]),
])
def test_attention_split(dev, hq, hkv, d, requests, window, sinks):
    print(f"[paged] split {hq}/{hkv} D={d} {requests} window {window}", flush=True)
    Step(dev, requests, hq, hkv, d, 16, window, sinks, seed=11).run()


def test_attention_more_requests_than_lanes(dev):
    rng = np.random.default_rng(8)
    Step(dev, [(int(x), 1) for x in rng.integers(1, 200, 300)], 16, 8, 64, 8, seed=8).run()


def test_attention_more_tokens_than_keys(dev):
    """Rows before position 0 see nothing and give 0."""
    st = Step(dev, [(64, 4), (33, 33)], 8, 2, 128, 16)
    st.seq_lens.copy_(ints([2, 33], dev))
    st.make_plan()
    st.attend()
    H.sync()
    got = st.o.cpu().double()
    assert (got[:2] == 0).all()
    k, v = (x[:2].double() for x in st.kv[0])
    o, away, size = PO.attention(st.q[2:4].double(), k, v, 0, 0)
    assert ((got[2:4] - o).abs() <= 2.0 ** -8 * (away + o.abs()) * 1.02 + 2.0 ** -12 * size).all()


def test_attention_large_scores(dev):
    """Scores of several hundred: the running reference moves, and rows whose
    largest score comes first keep it."""
    for seed in range(3):
        Step(dev, [(300, 1), (200, 200), (1500, 20)], 8, 2, 128, 16, std=60.0, seed=seed).run()


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (8, 2, 64), (16, 1, 128), (2, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_attention_nonfinite_hidden(dev, hq, hkv, d, window, sinks):
    """Infinities and NaN in keys and values reach exactly the rows that see
    them."""
    requests = [(200, 120), (90, 20), (70, 1)]
    st = Step(dev, requests, hq, hkv, d, 16, window, sinks, seed=2)
    bad = {(0, 150): float("nan"), (0, 90): float("inf"), (1, 80): -float("inf"),
           (2, 10): float("nan")}
    for (b, j), x in bad.items():
        page = int(st.table[b, j // 16])
        st.v[page, j % 16] = x
        st.k[page, j % 16, :, 0] = x
    st.run_unchecked = st.make_plan(), st.attend()
    H.sync()
    got = st.o.cpu().double()
    for b, (length, n) in enumerate(requests):
        seen = PO.visible(n, length, window, sinks)
        touched = np.zeros(n, bool)
        for (rb, j) in bad:
            if rb == b:
                touched |= seen[:, j]
        o, away, size = st.expect(b)
        g = got[st.start[b]:st.start[b + 1]]
        clean = torch.from_numpy(~touched)
        bound = 2.0 ** -8 * (away + o.abs()) * (1 + 2.0 ** -6) + 2.0 ** -12 * size
        assert ((g - o).abs() <= bound)[clean].all(), b
        assert not torch.isfinite(g[~clean]).any(), b


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (8, 2, 64), (16, 1, 128), (2, 1, 128)])
def test_attention_infinite_values_seen(dev, hq, hkv, d):
    """An infinite value gives infinity to the rows that see it, nothing to
    the others of its tile."""
    st = Step(dev, [(200, 120)], hq, hkv, d, 16, seed=4)
    for j, x in ((140, float("inf")), (170, -float("inf"))):
        st.v[int(st.table[0, j // 16]), j % 16, :, 5 if x > 0 else 70 % d] = x
    st.make_plan()
    st.attend()
    H.sync()
    got, first = st.o.cpu().double()[:120], 80
    o, away, size = st.expect(0)
    ok = (got - o).abs() <= 2.0 ** -8 * (away + o.abs()) * (1 + 2.0 ** -6) + 2.0 ** -12 * size
    rows = torch.arange(120)[:, None, None]
    dim = torch.arange(d)[None, None, :]
    plus, minus = (rows >= 140 - first) & (dim == 5), (rows >= 170 - first) & (dim == 70 % d)
    assert (got[plus.expand_as(got)] == float("inf")).all()
    assert (got[minus.expand_as(got)] == -float("inf")).all()
    assert ok[~(plus | minus).expand_as(got)].all()


def test_attention_other_plan(dev):
    """A plan made for other sizes: NaN everywhere, not a guess."""
    st = Step(dev, [(40, 1), (90, 3)], 8, 2, 128, 16)
    attn.paged_attention_plan(st.query_start, st.seq_lens, st.batch, st.rows, st.ps, st.blocks, 5,
                              0, st.hq, st.hkv, st.d, st.plan)
    st.attend()
    H.sync()
    assert torch.isnan(st.o).all()


def test_attention_arrays_of_any_content(dev):
    """Lengths and pages that are none: no access outside the tensors (the
    results are unspecified), and the next good step is right."""
    st = Step(dev, [(40, 1), (90, 30), (64, 2)], 8, 2, 128, 16)
    good = st.query_start.clone(), st.seq_lens.clone(), st.table.clone()
    for qs, lens in (([0, 4000000000, 5, 33], [7, 8, 9]), ([9, 3, 30, 1], [4000000000] * 3),
                     ([0, 36, 0, 36], [90, 90, 90])):
        st.query_start.copy_(ints(qs, dev))
        st.seq_lens.copy_(ints(lens, dev))
        st.table.fill_(-5)
        st.make_plan()
        st.attend()
        H.sync()
    for t, x in zip((st.query_start, st.seq_lens, st.table), good):
        t.copy_(x)
    st.o.fill_(3.0)
    st.run()


def test_attention_repeats_bit_for_bit(dev):
    st = Step(dev, [(3000, 1), (500, 200), (900, 30)], 16, 8, 128, 16)
    st.run()
    first = st.o.clone()
    for _ in range(3):
        st.o.fill_(3.0)
        st.make_plan()
        st.attend()
        assert torch.equal(st.o, first)


def test_attention_graph_and_streams(dev):
    """A captured step (plan and attention) replayed with other lengths, beside
    eager work, and a step on another stream with a plan and a workspace of its
    own at the same time."""
    steps = [Step(dev, [(x, 1), (y, 40), (300, 2)], 8, 2, 128, 16, seed=9) for x, y in
             ((700, 300),)]
    st = steps[0]
    other = Step(dev, [(1000, 33)], 16, 8, 128, 16, seed=10)
    st.run()
    other.run()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        st.make_plan(stream)
        st.attend(stream)
    for lens in ([700, 300, 300], [65, 41, 2], [700, 299, 64]):
        st.seq_lens.copy_(ints(lens, dev))
        st.o.fill_(3.0)
        other.o.fill_(3.0)
        H.sync()
        graph.replay()
        other.make_plan()
        other.attend()
        H.sync()
        other.check()
        got = st.o.cpu().double()
        for b, (length, n) in enumerate(zip(lens, (1, 40, 2))):
            k, v = (x[:length].double() for x in st.kv[b])
            o, away, size = PO.attention(st.q[st.start[b]:st.start[b + 1]].double(), k, v, 0, 0)
            g = got[st.start[b]:st.start[b + 1]]
            assert ((g - o).abs() <= 2.0 ** -8 * (away + o.abs()) * 1.02 + 2.0 ** -12 * size).all()
        st.o.fill_(3.0)
        st.make_plan()
        st.attend()
        H.sync()
        assert torch.equal(st.o.cpu().double(), got)


def test_tables_idle_requests_are_not_refused(dev):
    """Requests without new tokens, the padding of a batch, behind one whose rows
    do not fit: one is refused."""
    context, new = [0, 0, 0, 40, 7], [9, 9, 9, 0, 0]
    out = [ints([0] * 24, dev) for _ in range(5)]
    bt = ints(np.zeros((5, 8)), dev)
    attn.paged_tables_u32(ints(context, dev), ints(new, dev), 5, ints(range(20), dev), 20,
                          ints([20], dev), 8, bt, 8, 20, *out)
    H.sync()
    start, seq, pos, slots, status = (host(t) for t in out)
    assert start[:6] == [0, 9, 18, 27, 27, 27] and seq[:5] == [9, 9, 0, 40, 7]
    assert status[:2] == [16, 1]
    assert pos[:20] == [*range(9), *range(9), 0, 1] and slots[18:20] == [0xFFFFFFFF] * 2
