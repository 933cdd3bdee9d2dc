"""The 8-bit paged cache on the GPU.

V's codes and scales have to be the oracle's bit for bit: a value is bf16, its
code the nearest.  K's are those of the normalised and rotated values: most tests
let these be off by 2^-16 of the rotation's products, so the scale is the one of a
largest value inside that error, a code off by half a step more, 2^-4 of the value or
2^-10 of the scale; one asks for the codes bit for bit.  Reading back is exact.

Keys and values enter the attention's products without a rounding of their own,
so its bounds are those of the bf16 cache over the values that the codes stand
for.
"""
import numpy as np
import pytest
import torch

from tests import fp8_oracle as F8
from tests import helpers as H
from tests import paged_oracle as PO
from tests.test_paged_gpu import BATCHES, HEADS, Step, host, ints
from tests.test_paged_step_gpu import (EARLY, FORMS, SPOILT, Early, Wide, check_nan, check_rows,
                                       shape_of, wide_attention)
from toyinfer_amd import attn

pytestmark = pytest.mark.gpu

POSITIONS = 97


def bf16(x):
    return torch.from_numpy(np.asarray(x, np.float64)).to(torch.bfloat16)


# ------------------------------------------------------------------- write

class Writer:
    """K and V caches on the GPU beside the oracle's, and calls that go to both."""

    def __init__(self, dev, pages, ps, hq, hkv, d, seed=0, apart=0, interleaved=False):
        self.dev, self.pages, self.ps, self.hq, self.hkv, self.d = dev, pages, ps, hq, hkv, d
        self.rng = np.random.default_rng(seed)
        page = F8.page_bytes(ps, hkv, d) + apart
        self.k, self.v = (F8.Cache(pages, ps, hkv, d, page) for _ in range(2))
        if interleaved:
            both = torch.from_numpy(np.stack([self.k.raw, self.v.raw], 1)).to(dev)
            self.k_d, self.v_d = both[:, 0], both[:, 1]
        else:
            self.k_d, self.v_d = (torch.from_numpy(c.raw.copy()).to(dev) for c in (self.k, self.v))
        self.qw, self.kw = (bf16(self.rng.uniform(0.5, 1.5, d)) for _ in range(2))
        self.rope = torch.from_numpy(self.rng.uniform(-1, 1, (POSITIONS, d // 2, 2))).float()

    def rows(self, t, std=1.0):
        return bf16(self.rng.standard_normal((t, self.hkv, self.d)) * std)

    def launch(self, q, k, v, pos, slots, q_out, stream=None):
        attn.paged_qkv_prologue_fp8(q, k, v, self.qw.to(self.dev), self.kw.to(self.dev),
                                    self.rope.to(self.dev), POSITIONS, pos, slots, slots.numel(),
                                    1e-6, q_out, self.k_d, self.v_d, self.pages, self.ps,
                                    self.k_d.stride(0), self.hq, self.hkv, self.d, stream)

    def write(self, slots, k=None, v=None):
        """One call, checked against the oracle's."""
        t, hkv, d = len(slots), self.hkv, self.d
        slots = np.asarray(slots, np.uint32)
        k = self.rows(t, 3.0) if k is None else k
        v = self.rows(t) if v is None else v
        q = bf16(self.rng.standard_normal((t, self.hq, d)) * 2)
        pos = self.rng.integers(0, POSITIONS + 3, t)
        q_out = torch.empty_like(q, device=self.dev)
        self.launch(q.to(self.dev), k.to(self.dev), v.to(self.dev), ints(pos, self.dev),
                    ints(slots, self.dev), q_out)
        H.sync()
        cs = self.rope.double().numpy()[np.minimum(pos, POSITIONS - 1)]
        wide = np.abs(cs).sum(-1)

        def turned(x, w):
            x, w = x.double().numpy(), w.double().numpy()
            y = np.abs(PO.rms_rope(x, w, np.stack([np.ones_like(wide), np.zeros_like(wide)], -1), 1e-6))
            terms = np.tile((y[..., :d // 2] + y[..., d // 2:]) * wide[:, None], 2)
            return PO.rms_rope(x, w, cs, 1e-6), 2.0 ** -16 * terms

        exp, off = turned(q, self.qw)
        got = q_out.cpu().double().numpy()
        assert (np.abs(got - exp) <= 2.0 ** -8 * np.abs(exp) * 1.001 + off).all(), "q"
        self.v.write(slots, v.double().numpy())
        assert (self.v_d.cpu().numpy() == self.v.raw).all(), "V's bytes"
        self.check_k(slots, *turned(k, self.kw))

    def check_k(self, slots, x, off):
        now = F8.Cache(self.pages, self.ps, self.hkv, self.d, self.k.raw.shape[1])
        now.raw = self.k_d.cpu().numpy().copy()
        by_block = {}
        for t, s in enumerate(int(i) for i in slots):
            if s < self.pages * self.ps:
                by_block.setdefault(s // F8.BLOCK, []).append(t)
        exponents = {}
        for block, ts in by_block.items():
            page, b = divmod(block, self.ps // F8.BLOCK)
            opens = any(int(slots[t]) % F8.BLOCK == 0 for t in ts)
            for h in range(self.hkv):
                e = F8.POWERS[now.scale(page, h, b)]
                lo = F8.exponent_for(max((np.abs(x[t, h]) - off[t, h]).max() for t in ts))
                hi = F8.exponent_for(max((np.abs(x[t, h]) + off[t, h]).max() for t in ts))
                old = self.k.scale(page, h, b)
                if not opens and old in F8.POWERS:
                    lo, hi = max(lo, F8.POWERS[old]), max(hi, F8.POWERS[old])
                assert lo <= e <= hi, (block, h, lo, e, hi)
                exponents[block, h] = e
        live = [t for t, s in enumerate(slots) if s < self.pages * self.ps]
        for t in live:
            s = int(slots[t])
            e = np.array([exponents[s // F8.BLOCK, h] for h in range(self.hkv)])[:, None]
            half = np.maximum(2.0 ** -4 * (np.abs(x[t]) + off[t]), 2.0 ** (e - 10.0))
            assert (np.abs(now.row(s) - x[t]) <= half + off[t]).all(), ("K", t)
        # All other bytes: the oracle's, with these scales.
        self.k.write(slots, x, exponents)
        for t in live:
            page, r = divmod(int(slots[t]), self.ps)
            self.k.put_codes(page, r, now.codes()[page, :, r])
        assert (now.raw == self.k.raw).all(), "K's other bytes"


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (5, 1, 64), (12, 2, 64), (1, 1, 128), (6, 3, 128)])
@pytest.mark.parametrize("t", [1, 7, 16, 17, 130])
def test_write_prompt(dev, hq, hkv, d, t):
    """Prompts that begin at each kind of place in a block, into pages in any
    order, a row at the edge of a block and the last without a slot."""
    print(f"[fp8] write {hq}/{hkv} D={d} t={t}", flush=True)
    for first in (0, 3, 15):
        w = Writer(dev, t // 16 + 5, 16, hq, hkv, d, seed=t + first)
        pages = w.rng.permutation(w.pages)
        at = first + np.arange(t)
        slots = (pages[at // 16] * 16 + at % 16).astype(np.uint32)
        if t > 20:
            slots[32 - first], slots[t - 1] = 0xFFFFFFFF, w.pages * 16
        if first:
            w.write(pages[0] * 16 + np.arange(first))
        w.write(slots)


@pytest.mark.parametrize("ps", [16, 32, 256])
@pytest.mark.parametrize("d", [64, 128])
def test_write_steps(dev, ps, d):
    """Decoded tokens of 40 requests, values that grow and shrink from step to
    step: blocks grow, keep their scale and open, in pages further apart than
    they are long, K's beside V's."""
    w = Writer(dev, 40, ps, 4, 2, d, seed=ps, apart=48, interleaved=True)
    first = w.rng.integers(0, ps - 12, 40)
    w.write(np.concatenate([p * ps + f // 16 * 16 + np.arange(f % 16) for p, f in enumerate(first)]))
    for step, std in enumerate((1.0, 8.0, 0.01, 300.0, 1e4, 1.0, 3e-5)):
        slots = np.arange(40) * ps + first + step
        w.write(slots, v=w.rows(40, std), k=w.rows(40, std))


def test_write_drafted_tokens(dev):
    """Several tokens per request, rewritten from the middle of a block on, runs
    that cross the boundary of a wave's rows."""
    w = Writer(dev, 12, 16, 2, 2, 128, seed=2)
    w.write(np.concatenate([p * 16 + np.arange(9) for p in range(12)]))
    for start, n in ((9, 4), (10, 5), (3, 2), (9, 7)):
        w.write(np.concatenate([p * 16 + start + np.arange(n) for p in range(12)]), v=w.rows(12 * n, 2.0 ** n))
    w.write(np.concatenate([p * 16 + np.arange(16) for p in (3, 1)]))  # opens again


def test_write_rows_of_a_block_in_another_order(dev):
    """Neighbouring rows of one block need not ascend, nor leave no gaps."""
    w = Writer(dev, 4, 16, 2, 2, 64, seed=5)
    w.write(np.arange(16) + 16)
    w.write([31, 17, 25, 40, 33], v=w.rows(5, 50.0))
    w.write(np.arange(16)[::-1] + 48)


def test_write_values_at_the_edges(dev):
    """NaN, infinities, zeros, the largest and the smallest bf16, values at the
    borders of a scale and between two codes."""
    w = Writer(dev, 3, 16, 1, 1, 64, seed=1)
    v = np.zeros((12, 1, 64))
    v[1] = 3.3e38 * (1 - 2 * (np.arange(64) % 2))
    v[2, 0, :3] = np.inf, -np.inf, np.nan
    v[3] = 2.0 ** -133
    v[4], v[5, 0, 0], v[5, 0, 1:] = 448, 450, 2.0 ** -5 * np.arange(63)
    v[6] = np.arange(64) * 7.0
    w.write(np.arange(16, 17), v=bf16(v[:1]))          # zeros open a block
    for i in range(1, 12):
        w.write([16 + i], v=bf16(v[i:i + 1]))          # one after the other
    w.write(np.arange(32, 36), v=bf16(v[3:7]))
    w.write(np.arange(36, 40), v=bf16(v[8:12]))
    w.write([0], v=bf16(v[2:3]))


def test_write_many_tokens(dev):
    w = Writer(dev, 80, 64, 8, 4, 128, seed=9)
    pages = w.rng.permutation(80)
    at = np.arange(4000) + 500
    w.write((pages[at // 64] * 64 + at % 64).astype(np.uint32))


def test_write_rounds_exact_keys(dev):
    """Keys get the codes that their values in 64 bits round to: the kernel's are
    within 2^-48 of those, where one in 2^43 lies that close to a border."""
    w = Writer(dev, 40, 64, 4, 4, 128, seed=11)
    slots, pos = np.arange(2500) + 16, np.arange(2500) % POSITIONS
    q, k, v = (w.rows(2500, std) for std in (2.0, 3.0, 1.0))
    w.launch(q.to(dev), k.to(dev), v.to(dev), ints(pos, dev), ints(slots, dev), q.to(dev))
    H.sync()
    x = PO.rms_rope(k.double().numpy(), w.kw.double().numpy(), w.rope.double().numpy()[pos],
                    float(np.float32(1e-6)))
    w.k.write(slots, x)
    assert (w.k_d.cpu().numpy() == w.k.raw).all()


def test_write_in_place_and_again(dev):
    """q_out may be q, and a call gives the same bytes every time."""
    w = Writer(dev, 9, 16, 4, 2, 128)
    slots = np.arange(100) + 7
    q = bf16(w.rng.standard_normal((100, 4, 128))).to(dev)
    k, v, pos = w.rows(100).to(dev), w.rows(100).to(dev), ints(np.arange(100) % POSITIONS, dev)
    res = []
    for i in range(4):
        w.k_d.fill_(255)
        w.v_d.fill_(255)
        mine = q.clone()
        out = mine if i % 2 else torch.empty_like(q)
        w.launch(mine, k, v, pos, ints(slots, dev), out)
        res.append((out, w.k_d.clone(), w.v_d.clone()))
    H.sync()
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))


def test_write_same_slot_twice(dev):
    """Tokens that share a slot spoil no other block."""
    w = Writer(dev, 6, 16, 2, 2, 128, seed=3)
    before = w.k_d.clone()
    slots = np.concatenate([np.full(50, 20), [33, 33, 34], np.arange(48, 52)]).astype(np.uint32)
    t = len(slots)
    q = bf16(w.rng.standard_normal((t, 2, 128))).to(dev)
    v = w.rows(t)
    w.launch(q, w.rows(t).to(dev), v.to(dev), ints(np.arange(t), dev), ints(slots, dev), torch.empty_like(q))
    H.sync()
    for page in (0, 4, 5):
        assert torch.equal(w.k_d[page], before[page])
    w.v.write(np.arange(48, 52), v[-4:].double().numpy())
    assert (w.v_d[3].cpu().numpy() == w.v.raw[3]).all()


# -------------------------------------------------------------------- read

def read_back(dev, k, v, table, start, lens, rows, ps, blocks, hkv, d, fill=5.0):
    out = [torch.full((rows, hkv, d), fill, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    attn.paged_kv_read_fp8(k, v, table, ints(start, dev), ints(lens, dev), len(lens), rows, *out,
                           k.shape[0], ps, k.stride(0), blocks, hkv, d)
    H.sync()
    return [x.cpu() for x in out]


@pytest.mark.parametrize("hkv,d,ps", [(8, 128, 16), (1, 64, 16), (3, 64, 128), (5, 128, 32)])
def test_read(dev, hkv, d, ps):
    """Every code under scales of every size, contexts of any length, the last
    tokens of others, more of them than there are, rows behind the last."""
    rng = np.random.default_rng(ps + d)
    lens, news = [1, 200, 17, 0, 64, 333, 5], [1, 30, 17, 0, 64, 333, 9]
    need = [-(-x // ps) for x in lens]
    pages, blocks = sum(need) + 1, max(need) + 1
    caches = []
    for _ in range(2):
        c = F8.Cache(pages, ps, hkv, d)
        c.raw[:] = rng.integers(0, 256, c.raw.shape)
        for p in range(pages):
            for h in range(hkv):
                for b in range(ps // 16):
                    c.put_scale(p, h, b, 2.0 ** rng.integers(F8.LOW, F8.HIGH + 1))
        caches.append(c)
    order, table, at = rng.permutation(pages), np.full((len(lens), blocks), 0xFFFFFFFF, np.uint32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(news)])
    got = read_back(dev, *(torch.from_numpy(c.raw).to(dev) for c in caches), ints(table, dev), start,
                    lens, int(start[-1]) + 4, ps, blocks, hkv, d)
    for g, c in zip(got, caches):
        g = g.double().numpy()
        assert (g[start[-1]:] == 5).all()
        for b, (length, n) in enumerate(zip(lens, news)):
            for i in range(n):
                j = length - n + i
                row = g[start[b] + i]
                if j < 0:
                    assert (row == 0).all()
                else:
                    want = c.row(int(table[b, j // ps]) * ps + j % ps)
                    assert np.array_equal(row, want, equal_nan=True), (b, j)


@pytest.mark.parametrize("batch", [1, 2, 255, 4096])
def test_read_batches(dev, batch):
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 5, batch)
    w = Writer(dev, batch, 16, 1, 1, 64, seed=batch)
    slots = np.concatenate([b * 16 + np.arange(n) for b, n in enumerate(lens)] + [np.zeros(0)]).astype(np.uint32)
    slots = slots if len(slots) else np.array([0], np.uint32)
    if len(slots) < 3000:
        w.write(slots)
    else:
        k = w.rows(len(slots)).to(dev)
        w.launch(torch.zeros(len(slots), 1, 64, dtype=torch.bfloat16, device=dev), k, k,
                 ints(slots % 16, dev), ints(slots, dev),
                 torch.empty(len(slots), 1, 64, dtype=torch.bfloat16, device=dev))
        H.sync()
        w.v.raw = w.v_d.cpu().numpy()
    start = np.concatenate([[0], np.cumsum(lens)])
    _, v = read_back(dev, w.k_d, w.v_d, ints(np.arange(batch)[:, None], dev), start, lens,
                     int(start[-1]) + 1, 16, 1, 1, 64)
    want = np.stack([w.v.row(b * 16 + i) for b, n in enumerate(lens) for i in range(n)] + [np.full((1, 64), 5.0)])
    assert np.array_equal(v.double().numpy(), want)


def test_read_arrays_of_any_content(dev):
    """Lengths and pages that are none: no access outside the tensors."""
    w = Writer(dev, 4, 16, 2, 2, 64)
    w.write(np.arange(64))
    for start, lens in (([0, 4000000000, 5, 33], [7, 8, 9]), ([9, 3, 30, 1], [4000000000] * 3),
                        ([0, 36, 0, 36], [90, 90, 90]), ([50, 60, 70, 80], [1, 2, 3])):
        read_back(dev, w.k_d, w.v_d, ints(np.full((3, 4), 0xFFFFFFFB), dev), start, lens, 36, 16, 4, 2, 64)


# --------------------------------------------------------------- attention

class In8Bits:
    """A Step's requests in 8-bit caches whose unwritten rows, blocks and pages
    are NaN; `kv` becomes what the codes stand for."""

    apart = 0

    def __init__(self, *args, interleaved=False, **kw):
        super().__init__(*args, **kw)
        hkv, d, ps = self.hkv, self.d, self.ps
        n = F8.page_bytes(ps, hkv, d) + self.apart
        both = torch.full((self.pages, 2, n), 255, dtype=torch.uint8)
        codes = both[:, :, :hkv * ps * d].view(self.pages, 2, hkv, ps, d)
        at = hkv * ps * d
        scales = both[:, :, at:at + hkv * ps // 16 * 4].view(torch.float32).view(self.pages, 2, hkv, ps // 16)
        table = self.table.cpu().numpy()
        held = []
        for b, kv in enumerate(self.kv):
            new = []
            for which, x in enumerate(kv):
                rows = x.shape[0]
                wide = torch.zeros(-(-rows // 16) * 16, hkv, d)
                wide[:rows] = x.float() * torch.exp2(torch.arange(rows) % 5 - 2.0)[:, None, None]
                blocks = wide.view(-1, 16, hkv, d)
                most = blocks.abs().amax((1, 3))
                m, e = torch.frexp(most)
                s = torch.ldexp(torch.ones_like(most), e - 9 + (m > 0.875).int())
                c = (blocks / s[:, None, :, None]).to(torch.float8_e4m3fn)
                new.append((c.float() * s[:, None, :, None]).view(-1, hkv, d)[:rows].to(torch.bfloat16))
                c = c.view(torch.uint8).view(-1, hkv, d)
                for j in range(-(-rows // ps)):
                    page, m = int(table[b, j]), min(ps, rows - j * ps)
                    codes[page, which, :, :m] = c[j * ps:j * ps + m].transpose(0, 1)
                    mb = -(-m // 16)
                    scales[page, which, :, :mb] = s[j * ps // 16:j * ps // 16 + mb].t()
            held.append(tuple(new))
        self.kv = held
        del self.k, self.v
        if interleaved:
            both = both.to(self.dev)
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k, self.v = (both[:, i].contiguous().to(self.dev) for i in range(2))
        self.stride = self.k.stride(0)

    def attend(self, stream=None):
        attn.paged_attention_fp8(self.q_d, self.k, self.v, self.o, self.table, self.plan,
                                 self.batch, self.rows, self.pages, self.ps, self.stride,
                                 self.blocks, self.window, self.sinks, self.hq, self.hkv, self.d,
                                 self.ws, stream)

    def put(self, which, b, j, dim, code):
        """`code` at a key and dim of every head."""
        cache = (self.k, self.v)[which]
        at = torch.arange(self.hkv, device=self.dev) * self.ps * self.d + j % self.ps * self.d + dim
        cache[int(self.table[b, j // self.ps]), at] = code


class Step8(In8Bits, Step):
    pass


class Wide8(In8Bits, Wide):
    pass


class Early8(In8Bits, Early):
    pass


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("name", BATCHES)
def test_attention(dev, name, hq, hkv, d):
    print(f"[fp8] attention {name} {hq}/{hkv} D={d}", flush=True)
    Step8(dev, BATCHES[name], hq, hkv, d, 16, seed=hq + d).run()


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 512])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_page_sizes(dev, ps, d):
    Step8(dev, [(700, 1), (130, 130), (333, 40), (64, 2), (1, 1)], 8, 2, d, ps, seed=ps,
          interleaved=True).run()


@pytest.mark.parametrize("ps,apart", [(16, 16), (16, 96), (64, 48), (4096, 0), (16384, 112)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_strides(dev, ps, apart, d):
    """Pages at any multiple of 16 bytes, and large ones."""
    class Spread(Step8):
        pass
    Spread.apart = apart
    Spread(dev, [(700, 1), (130, 130), (5000, 40), (64, 2), (1, 1)], 8, 2, d, ps, seed=ps).run()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (64, 0), (100, 70), (300, 4),
                                          (5000, 3)])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (6, 2, 64)])
def test_attention_window(dev, window, sinks, hq, hkv, d):
    print(f"[fp8] window {window} sinks {sinks} {hq}/{hkv}", flush=True)
    Step8(dev, [(900, 1), (150, 150), (500, 60), (64, 3), (1, 1)], hq, hkv, d, 32, window, sinks,
          seed=window).run()


@pytest.mark.parametrize("case", range(len(FORMS)))
def test_each_form(dev, case):
    """Units of every size, whole and in pieces (the plan and so the forms are
    those of the bf16 cache)."""
    hq, hkv, d, requests = FORMS[case]
    st = Wide8(dev, requests, hq, hkv, d, 16, seed=case)
    st.make_plan()
    H.sync()
    print(f"[fp8] {hq}/{hkv} D={d} {requests[:3]}: {shape_of(st)}", flush=True)
    st.run()


@pytest.mark.parametrize("hq,hkv,d,requests", [
    (64, 1, 128, [(700, 3), (90, 90)]),
    (71, 1, 64, [(500, 2), (40, 40)]),
    (9, 3, 128, [(3000, 1), (260, 130)]),
    (260, 260, 64, [(200, 1), (70, 20)]),
    (25, 5, 128, [(2042, 373)]),
    (8, 8, 128, [(6000, 200)]),
])
def test_head_layouts(dev, hq, hkv, d, requests):
    print(f"[fp8] heads {hq}/{hkv} D={d}", flush=True)
    Wide8(dev, requests, hq, hkv, d, 16, seed=hq).run()


@pytest.mark.parametrize("window,sinks", [(0, 0), (9000, 100)])
@pytest.mark.parametrize("ps", [16, 64, 256])
def test_long_contexts(dev, ps, window, sinks):
    print(f"[fp8] long, page size {ps} window {window}", flush=True)
    Wide8(dev, [(40001, 1), (20000, 100), (33000, 9)], 8, 2, 128, ps, window, sinks, seed=ps).run()


def test_many_requests(dev):
    rng = np.random.default_rng(4)
    Wide8(dev, [(int(x), 1) for x in rng.integers(1, 700, 1000)], 16, 4, 128, 16, seed=4).run()


@pytest.mark.parametrize("window,sinks", [(0, 0), (37, 2), (1 << 31, 5)])
@pytest.mark.parametrize("case", range(len(EARLY)))
def test_rows_on_both_sides_of_position_0(dev, case, window, sinks):
    hq, hkv, d, requests = EARLY[case]
    print(f"[fp8] before 0: {hq}/{hkv} D={d} {requests[:4]} window {window}", flush=True)
    Early8(dev, requests, hq, hkv, d, 16, window, sinks, seed=case).run()


@pytest.mark.parametrize("case", range(len(SPOILT)))
def test_codes_that_are_nan(dev, case):
    """A NaN in V reaches the dims of the rows that see it, and no others; one in
    K the rows that see it."""
    hq, hkv, d, requests, window, sinks, at = SPOILT[case]
    st = Wide8(dev, requests, hq, hkv, d, 16, window, sinks, seed=case)
    st.make_plan()
    H.sync()
    print(f"[fp8] NaN: {hq}/{hkv} D={d} {requests[:3]}: {shape_of(st)}", flush=True)
    st.run()
    for i, (b, j, dim, _) in enumerate(at):
        st.put(1, b, j, dim, 127 + 128 * (i % 2))
    for _ in range(2):
        st.o.fill_(3.0)
        st.attend()
        H.sync()
        check_nan(st, at)
    b, j, dim, _ = at[0]
    st.put(0, b, j, dim, 255)
    st.attend()
    H.sync()
    length, n = requests[b]
    seen = torch.from_numpy(PO.visible(n, length, window, sinks))[:, j]
    got = st.o[int(st.start[b]):int(st.start[b + 1])].cpu()
    assert torch.isnan(got[seen]).all()
    other = (dim + 1) % d  # (no NaN of V in it, or in rows that see it only)
    if all(x[2] != other for x in at):
        assert torch.isfinite(got[~seen][..., other]).all()


@pytest.mark.parametrize("hq,d,requests", [(32, 64, [(5000, 5000), (900, 1)])])
def test_more_spoilt_blocks_than_marks(dev, hq, d, requests):
    st = Wide8(dev, requests, hq, hq, d, 16, seed=3)
    at = [(0, j, 11, None) for j in range(3, requests[0][0], 7)]
    for b, j, dim, _ in at:
        st.put(1, b, j, dim, 127)
    st.make_plan()
    st.attend()
    H.sync()
    assert shape_of(st)[1]
    check_nan(st, at)


def test_hidden_scales_that_are_none(dev):
    """Scales of blocks that no row sees, behind a window and past the last key,
    may hold anything."""
    for requests, window in (([(700, 1), (300, 40)], 100), ([(330, 330)], 64), ([(129, 1), (65, 3)], 0)):
        for d in (64, 128):
            st = Step8(dev, requests, 8, 2, d, 64, window, 0, seed=d)
            at = 2 * 64 * d
            scales = st.v[:, at:at + 32].view(torch.float32).view(-1, 2, 4)
            for b, (length, n) in enumerate(requests):
                low = max(0, length - n + 1 - window) if window else 0
                for block in range(low // 16):
                    scales[int(st.table[b, block // 4]), :, block % 4] = (float("inf"), float("nan"))[block % 2]
            st.run()


def test_attention_other_plan(dev):
    st = Step8(dev, [(40, 1), (90, 3)], 8, 2, 128, 16)
    attn.paged_attention_plan(st.query_start, st.seq_lens, st.batch, st.rows, st.ps, st.blocks, 5,
                              0, st.hq, st.hkv, st.d, st.plan)
    st.attend()
    H.sync()
    assert torch.isnan(st.o).all()


def test_attention_arrays_of_any_content(dev):
    st = Step8(dev, [(40, 1), (90, 30), (64, 2)], 8, 2, 128, 16)
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


def test_attention_large_scores(dev):
    for seed in range(3):
        Step8(dev, [(300, 1), (200, 200), (1500, 20)], 8, 2, 128, 16, std=60.0, seed=seed).run()


def test_no_new_tokens(dev):
    st = Step8(dev, [(40, 0), (0, 0), (300, 0)], 8, 2, 128, 16)
    st.run()
    assert (st.o == 3.0).all() and not st.ws[:4 * (st.hkv + 2)].any()


def test_attention_repeats_bit_for_bit(dev):
    st = Step8(dev, [(3000, 1), (500, 200), (900, 30)], 16, 8, 128, 16)
    st.run()
    first = st.o.clone()
    for _ in range(3):
        st.o.fill_(3.0)
        st.make_plan()
        st.attend()
        assert torch.equal(st.o, first)


def test_long_contexts_miss_no_tile(dev):
    """As over the bf16 cache: the RMS over a request's elements sees a tile that
    the elements' bound cannot."""
    rms = lambda x: x.square().mean().sqrt().item()
    for d in (64, 128):
        st = Wide8(dev, [(40001, 1), (20000, 33), (33000, 9)], 8, 2, d, 16, 0, 0, seed=d)
        st.run()
        for b, (length, n) in enumerate(st.requests):
            rows = slice(int(st.start[b]), int(st.start[b + 1]))
            k, v = (x.to(dev) for x in st.kv[b])
            o, _ = wide_attention(st.q_d[rows], k, v, 0, 0)
            error = rms(st.o[rows].double() - o) / rms(o)
            print(f"[fp8] {length} keys, D={d}: RMS {error:.5f}", flush=True)
            assert error < 2.0 ** -7, b


def test_equals_the_bf16_cache(dev):
    """Units of more than 32 rows run the same products over the same operands:
    bit for bit what the bf16 cache of the values gives."""
    for hq, hkv, d, requests, window in ((32, 8, 128, [(2048, 2048)], 0), (8, 8, 128, [(6000, 1000)], 900),
                                         (32, 8, 64, [(1500, 1400)] * 3, 0)):
        st = Wide8(dev, requests, hq, hkv, d, 64, window, 4 if window else 0, seed=7)
        st.run()
        pages = torch.zeros(2, st.pages, 64, hkv, d, dtype=torch.bfloat16)
        table = st.table.cpu().numpy()
        for b, kv in enumerate(st.kv):
            for which, x in enumerate(kv):
                for j in range(0, x.shape[0], 64):
                    part = x[j:j + 64]
                    pages[which, int(table[b, j // 64]), :part.shape[0]] = part
        o = torch.full_like(st.o, 3.0)
        k, v = (p.contiguous().to(dev) for p in pages)
        attn.paged_attention_bf16(st.q_d, k, v, o, st.table, st.plan, st.batch, st.rows, st.pages, 64,
                                  64 * hkv * d, st.blocks, st.window, st.sinks, hq, hkv, d, st.ws)
        H.sync()
        # (Others stream their keys, whose dims are summed in another order.)
        raw = st.plan.cpu().numpy()
        head = raw[:256].view(np.uint32)
        every = raw[256:256 + 48 * int(head[10] + head[12])].view(np.uint32).reshape(-1, 12)
        same = torch.zeros(st.rows, hq, dtype=torch.bool)
        group = hq // hkv
        for it in every:
            if 32 < it[3] <= 256 and it[0] < st.batch:
                for row in range(int(it[2]), int(it[2] + it[3])):
                    same[int(it[1]) + row // group, row % group::group] = True
        print(f"[fp8] {requests[:2]}: {shape_of(st)}, {same.float().mean():.2f} of the rows", flush=True)
        assert same.float().mean() > 0.8
        assert torch.equal(o[same.to(dev)], st.o[same.to(dev)])


def test_pages_past_4_gib(dev):
    """Byte offsets beyond 32 bits in the write's slots, the read's and the
    attention's pages."""
    hq, hkv, d, ps = 8, 4, 128, 64
    page = attn.paged_fp8_page_bytes(ps, hkv, d)
    pages = (2 ** 32 + 2 ** 28) // page
    kc, vc = (torch.empty(pages, page, dtype=torch.uint8, device=dev) for _ in range(2))
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
    print("[fp8] write past 4 GiB", flush=True)
    attn.paged_qkv_prologue_fp8(q, k, v, one, one, rope, length, ints(range(length), dev),
                                ints(slots, dev), length, 1e-6, q_out, kc, vc, pages, ps, page, hq,
                                hkv, d)
    H.sync()
    rows_k, rows_v = (x.to(dev) for x in read_back(dev, kc, vc, ints([table], dev), [0, length], [length],
                                                   length, ps, 5, hkv, d))
    small = F8.Cache(5, ps, hkv, d)
    small.write(np.arange(length), v.cpu().double().numpy())
    assert np.array_equal(rows_v.cpu().double().numpy(), np.stack([small.row(j) for j in range(length)]))
    qn = q_out[length - new:].contiguous()
    for n in (new, 1):
        o = torch.empty_like(qn[:n])
        plan = attn.paged_attention_plan_buffer(1, n, hq, hkv, d, dev)
        ws = attn.paged_attention_workspace(hq, hkv, d, dev)
        print("[fp8] attention past 4 GiB", flush=True)
        attn.paged_attention_plan(ints([0, n], dev), ints([length], dev), 1, n, ps, 5, 0, 0, hq, hkv,
                                  d, plan)
        attn.paged_attention_fp8(qn[new - n:].contiguous(), kc, vc, o, ints(table, dev), plan, 1, n,
                                 pages, ps, page, 5, 0, 0, hq, hkv, d, ws)
        H.sync()
        check_rows(o, qn[new - n:], rows_k, rows_v, 0, 0, "past 4 GiB")


# ------------------------------------------------------- operators together

class Server8:
    """A tiny serving loop over the tables, the plan and the 8-bit operators:
    requests with prompts of their own, taken in chunks, then decoded; random q, k,
    v per step.  V's bytes are the oracle's after every step; what the caches hold
    is read back, and the attention checked over that."""

    def __init__(self, dev, prompts, hq, hkv, d, ps, window, sinks, rows, seed):
        self.dev, self.hq, self.hkv, self.d, self.ps = dev, hq, hkv, d, ps
        self.window, self.sinks, self.rows = window, sinks, rows
        self.batch, self.blocks, self.pages = len(prompts), 48, 160
        self.left, self.lens = list(prompts), [0] * len(prompts)
        g = torch.Generator().manual_seed(seed)
        self.bf = lambda *shape, std=1.0: (torch.randn(shape, generator=g) * std).to(torch.bfloat16).to(dev)
        self.v_now = F8.Cache(self.pages, ps, hkv, d)
        self.kc, self.vc = (torch.from_numpy(self.v_now.raw.copy()).to(dev) for _ in range(2))
        self.qw, self.kw = self.bf(d), self.bf(d)
        ang = torch.rand(700, d // 2, generator=g) * 6.28
        self.rope = torch.stack([ang.cos(), ang.sin()], -1).float().to(dev)
        order = np.random.default_rng(seed).permutation(self.pages)
        self.free_d, self.num_free = ints(order, dev), ints([self.pages], dev)
        self.table = ints(np.zeros((self.batch, self.blocks)), dev)
        self.ctx, self.new = ints([0] * self.batch, dev), ints([0] * self.batch, dev)
        self.query_start, self.all_start = (ints([0] * (self.batch + 1), dev) for _ in range(2))
        self.seq_lens = ints([0] * self.batch, dev)
        self.positions, self.slots = ints([0] * rows, dev), ints([0] * rows, dev)
        self.status = ints([0, 0], dev)
        self.q, self.k, self.v = self.bf(rows, hq, d), self.bf(rows, hkv, d), self.bf(rows, hkv, d)
        self.q_out, self.o = torch.empty_like(self.q), torch.empty_like(self.q)
        self.back = sum(prompts) + 20 * self.batch
        self.k_out, self.v_out = (torch.empty(self.back, hkv, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
        self.plan = attn.paged_attention_plan_buffer(self.batch, rows, hq, hkv, d, dev)
        self.ws = attn.paged_attention_workspace(hq, hkv, d, dev)
        self.keys = [torch.zeros(0, hkv, d, dtype=torch.float64) for _ in prompts]

    def launch(self, stream=None):
        """The whole step, and whole contexts read back: nothing of it depends on a
        length on the host."""
        attn.paged_tables_u32(self.ctx, self.new, self.batch, self.free_d, self.pages,
                              self.num_free, self.ps, self.table, self.blocks, self.rows,
                              self.query_start, self.seq_lens, self.positions, self.slots,
                              self.status, stream)
        attn.paged_attention_plan(self.query_start, self.seq_lens, self.batch, self.rows, self.ps,
                                  self.blocks, self.window, self.sinks, self.hq, self.hkv, self.d,
                                  self.plan, stream)
        attn.paged_qkv_prologue_fp8(self.q, self.k, self.v, self.qw, self.kw, self.rope, 700,
                                    self.positions, self.slots, self.rows, 1e-6, self.q_out,
                                    self.kc, self.vc, self.pages, self.ps, self.kc.stride(0),
                                    self.hq, self.hkv, self.d, stream)
        attn.paged_attention_fp8(self.q_out, self.kc, self.vc, self.o, self.table, self.plan,
                                 self.batch, self.rows, self.pages, self.ps, self.kc.stride(0),
                                 self.blocks, self.window, self.sinks, self.hq, self.hkv, self.d,
                                 self.ws, stream)
        attn.paged_kv_read_fp8(self.kc, self.vc, self.table, self.all_start, self.seq_lens,
                               self.batch, self.back, self.k_out, self.v_out, self.pages, self.ps,
                               self.kc.stride(0), self.blocks, self.hkv, self.d, stream)

    def step(self, chunk, launch):
        new = [min(chunk, x) if x else 1 for x in self.left]
        self.left = [x - n if x else 0 for x, n in zip(self.left, new)]
        self.ctx.copy_(ints(self.lens, self.dev))
        self.new.copy_(ints(new, self.dev))
        ends = [x + n for x, n in zip(self.lens, new)]
        self.all_start.copy_(ints(np.concatenate([[0], np.cumsum(ends)]), self.dev))
        std = float(2.0 ** np.random.default_rng(sum(ends)).integers(-3, 4))  # blocks grow now and then
        for t in (self.q, self.k, self.v):
            t.copy_(self.bf(*t.shape, std=std))
        for t in (self.o, self.k_out, self.v_out):
            t.fill_(3.0)
        H.sync()
        launch()
        H.sync()
        left, refused = host(self.status)
        assert refused == 0
        self.num_free.copy_(ints([left], self.dev))
        slots = np.array(host(self.slots), np.int64)
        self.v_now.write(slots, self.v.cpu().double().numpy())
        assert (self.vc.cpu().numpy() == self.v_now.raw).all()
        at = base = 0
        for b, n in enumerate(new):
            rows, before = slice(at, at + n), self.lens[b]
            self.lens[b] += n
            length, at = self.lens[b], at + n
            cs = self.rope[before:length].double().cpu().numpy()
            k = PO.rms_rope(self.k[rows].double().cpu().numpy(), self.kw.double().cpu().numpy(), cs, 1e-6)
            self.keys[b] = torch.cat([self.keys[b], torch.from_numpy(k)])
            got_k, got_v = (x[base:base + length] for x in (self.k_out, self.v_out))
            base += length
            # A block's scale may be set by its largest value, of any row and head dim:
            # a code is off by at most 2^-4 of the value or 2^-9 (with rows rounded again
            # below 2^-9 of all scales before it) of the largest / 224.
            most = torch.cat([self.keys[b].abs(), torch.zeros(-length % 16, self.hkv, self.d)]).view(
                -1, 16, self.hkv, self.d).amax((1, 3)).repeat_interleave(16, 0)[:length, :, None]
            off = 2.0 ** -4 * self.keys[b].abs() * 1.01 + 2.0 ** -8 * most / 224
            assert ((got_k.cpu().double() - self.keys[b]).abs() <= off).all(), b
            check_rows(self.o[rows], self.q_out[rows], got_k, got_v, self.window, self.sinks, b)
        assert (self.o[at:] == 3.0).all()
        assert (self.k_out[base:] == 3.0).all() and (self.v_out[base:] == 3.0).all()


@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 4)])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (6, 2, 64)])
def test_serving_steps(dev, hq, hkv, d, window, sinks):
    print(f"[fp8] serving {hq}/{hkv} D={d} window {window}", flush=True)
    s = Server8(dev, [130, 1, 300, 17, 64], hq, hkv, d, 16, window, sinks, 270, seed=hq + window)
    for _ in range(8):
        s.step(64, s.launch)


def test_serving_steps_captured(dev):
    """The same as one captured graph, replayed step after step with eager work
    between the replays."""
    s = Server8(dev, [100, 33, 200], 16, 8, 128, 32, 0, 0, 140, seed=5)
    s.step(40, s.launch)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        s.launch(stream)
    other = Step8(dev, [(700, 1), (90, 33)], 8, 2, 128, 16, seed=1)
    for _ in range(6):
        s.step(40, graph.replay)
        other.run()
    s.step(40, s.launch)


def test_caches_of_both_kinds_share_plan_and_workspace(dev):
    """Layers with a bf16 cache and layers with an 8-bit one in one step: one plan,
    one workspace, in turn."""
    requests = [(3000, 1), (500, 120), (60, 3), (900, 20)]
    wide, narrow = Step(dev, requests, 16, 8, 128, 16, seed=3), Step8(dev, requests, 16, 8, 128, 16, seed=3)
    narrow.plan, narrow.ws = wide.plan, wide.ws
    wide.make_plan()
    for _ in range(3):
        for st in (wide, narrow):
            st.o.fill_(3.0)
            st.attend()
    H.sync()
    wide.check()
    narrow.check()
    assert not wide.ws[:4 * (8 + 2)].any()


def test_graphs_that_share_a_workspace(dev):
    one = Step8(dev, [(700, 1), (300, 40), (900, 1)], 8, 2, 128, 16, seed=21)
    two = Step8(dev, [(3000, 1), (64, 64), (100, 5)], 8, 2, 128, 16, 70, 4, seed=22)
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
    st = Step8(dev, [(3000, 1), (500, 120), (60, 3)], 16, 8, 64, 16, seed=23)
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


@pytest.mark.parametrize("hq,hkv,d,requests", [
    (20, 1, 128, [(700, 1), (300, 1), (64, 1), (65, 1)]),        # 20 rows
    (32, 1, 64, [(9000, 1), (31, 1)]),                           # 32
    (6, 2, 128, [(700, 7), (5000, 10), (100, 5), (64, 6)]),      # 21, 30, 15, 18
    (17, 17, 64, [(900, 17), (500, 16), (700, 1), (300, 32)]),
    (4, 1, 128, [(700, 4), (300, 5), (1, 1), (2, 2), (65, 3)]),  # 16 and 20 rows
])
@pytest.mark.parametrize("window", [0, 130])
def test_streams_of_each_width(dev, hq, hkv, d, requests, window):
    """Streams of up to 16 rows and of 17 to 32, one after the other in a lane's
    list."""
    Step8(dev, requests, hq, hkv, d, 16, window, 3 if window else 0, seed=hq).run()


def test_decoded_tokens_keep_the_weights_precision(dev):
    """Streams of up to 16 rows round a weight twice (a bf16 value and what it
    leaves), so an element's RMS error is the output's own rounding: a step 2^-7 of
    the power of two below the value, over sqrt(12), against values whose mantissas
    spread over [1, 2): 2^-7 / sqrt(12 * 7 / 3) = 0.0015 of the RMS.  One part alone
    would add a weight's rounding, as much again in another direction (0.0021); the
    limit is 2^-9 = 0.00195."""
    st = Wide8(dev, [(5000, 1), (9000, 2), (3000, 4)], 32, 8, 128, 16, seed=5)
    st.run()
    rms = lambda x: x.square().mean().sqrt().item()
    for b in range(3):
        rows = slice(int(st.start[b]), int(st.start[b + 1]))
        k, v = (x.to(dev) for x in st.kv[b])
        o, _ = wide_attention(st.q_d[rows], k, v, 0, 0)
        assert rms(st.o[rows].double() - o) < 2.0 ** -9 * rms(o), b


def test_binding_refuses_on_the_gpu(dev):
    """Tensors of another type, size, layout or device: refused, nothing written."""
    st = Step8(dev, [(40, 1), (90, 3)], 8, 2, 128, 16)
    st.make_plan()
    H.sync()
    before = st.k.clone(), st.v.clone()

    def attend(**kw):
        a = dict(q=st.q_d, k=st.k, v=st.v, o=st.o, table=st.table, plan=st.plan, ws=st.ws)
        a.update(kw)
        attn.paged_attention_fp8(a["q"], a["k"], a["v"], a["o"], a["table"], a["plan"], st.batch,
                                 st.rows, st.pages, st.ps, st.stride, st.blocks, 0, 0, st.hq,
                                 st.hkv, st.d, a["ws"])

    for kw in (dict(q=st.q_d.half()), dict(q=st.q_d[:-1]), dict(q=st.q_d.cpu()), dict(k=st.k[1:]),
               dict(v=st.v.cpu()), dict(k=st.k.view(torch.int8)), dict(k=st.k.view(-1)),
               dict(k=st.k.view(torch.bfloat16)), dict(o=st.o.float()),
               dict(v=torch.cat([st.v, st.v], 1)[:, :st.v.shape[1]]), dict(table=st.table.long()),
               dict(table=st.table[:1]), dict(plan=st.plan[:-256]), dict(ws=st.ws[:-16]), dict(o=st.q_d)):
        with pytest.raises(attn.ToyInferError):
            attend(**kw)

    rows, new = st.rows, st.q_d[:, :2].contiguous()
    w, rope = torch.ones(128, dtype=torch.bfloat16, device=dev), torch.zeros(99, 64, 2, device=dev)
    index = torch.zeros(rows, dtype=torch.int32, device=dev)

    def write(**kw):
        a = dict(q=st.q_d, k=new, v=new, w=w, rope=rope, pos=index, slots=index, out=st.q_d, kc=st.k, vc=st.v)
        a.update(kw)
        attn.paged_qkv_prologue_fp8(a["q"], a["k"], a["v"], a["w"], a["w"], a["rope"], 99, a["pos"],
                                    a["slots"], rows, 1e-6, a["out"], a["kc"], a["vc"], st.pages,
                                    st.ps, st.stride, 8, 2, 128)

    for kw in (dict(k=new[1:]), dict(v=new.float()), dict(w=w[1:]), dict(rope=rope[1:]), dict(pos=index.long()),
               dict(slots=index[:1]), dict(kc=st.k[:, 16:]), dict(vc=st.k), dict(out=new), dict(kc=st.k.cpu())):
        with pytest.raises(attn.ToyInferError):
            write(**kw)

    outs = [torch.full((43, 2, 128), 3.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]

    def read(**kw):
        a = dict(k=st.k, v=st.v, table=st.table, start=st.query_start, lens=st.seq_lens, ko=outs[0], vo=outs[1])
        a.update(kw)
        attn.paged_kv_read_fp8(a["k"], a["v"], a["table"], a["start"], a["lens"], 2, 43, a["ko"], a["vo"],
                               st.pages, st.ps, st.stride, st.blocks, 2, 128)

    for kw in (dict(k=st.k[1:]), dict(table=st.table[:1]), dict(start=st.query_start[:2]), dict(lens=st.seq_lens.long()),
               dict(ko=outs[0][1:]), dict(vo=outs[0]), dict(ko=outs[0].half()), dict(v=st.v.cpu())):
        with pytest.raises(attn.ToyInferError):
            read(**kw)
    H.sync()
    assert (st.o == 3.0).all() and all((x == 3.0).all() for x in outs)
    assert torch.equal(st.k, before[0]) and torch.equal(st.v, before[1])
    attend()
    H.sync()
    st.check()
