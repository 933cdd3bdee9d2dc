"""Attention over the 8-bit paged cache where blocks that no row sees hold anything:
pages behind a window whose table entries are stale, or none, between the first
tokens kept in sight and the window, and blocks behind the last key.  Nothing of
them may reach a result, so the bounds are those of the cache without them."""
import numpy as np
import pytest
import torch

from tests.test_paged_fp8_gpu import Step8
from tests.test_paged_step_gpu import shape_of

pytestmark = pytest.mark.gpu

# Scales, most of them none that the writer makes: finite ones whose largest codes pass
# bf16's range, infinity and NaN, and small, negative and other ones.
SCALES = [2.0 ** 119, 2.0 ** 120, 2.0 ** 125, 2.0 ** 127, 3e38, -(2.0 ** 126), float("inf"), float("nan"),
          0.0, -0.0, 1e-40, 2.0 ** -126, -1.5, 0.7]


def spoil(st, scale):
    """`scale` and the largest codes, of either sign, into both caches' hidden blocks;
    returns how many."""
    hkv, d, ps = st.hkv, st.d, st.ps
    n = hkv * ps * d
    code = torch.where(torch.arange(d) % 3 == 0, 0xFE, 0x7E).to(torch.uint8).to(st.dev)
    views = [(c[:, :n].view(-1, hkv, ps, d), c[:, n:n + hkv * ps // 4].view(torch.float32).view(-1, hkv, ps // 16))
             for c in (st.k, st.v)]
    table, count = st.table.cpu().numpy(), 0
    for b, (length, new) in enumerate(st.requests):
        low = max(0, length - new + 1 - st.window) if st.window else 0
        for i in range(-(-length // ps) * ps // 16):
            behind = 16 * i + 15 < low and 16 * i >= st.sinks
            if behind or 16 * i >= length:
                page, at = int(table[b, 16 * i // ps]), 16 * i % ps
                for codes, scales in views:
                    codes[page, :, at:at + 16] = code
                    scales[page, :, at // 16] = scale
                count += behind
    return count


@pytest.mark.parametrize("window,sinks", [(100, 0), (100, 20), (37, 4)])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("hq,d", [(8, 64), (8, 128), (24, 128)])
def test_hidden_blocks_of_any_content(dev, hq, d, ps, window, sinks):
    """Units of up to 16 rows, of 17 to 32 and larger ones; each scale by itself."""
    # (Windows that begin inside a tile, two blocks or more behind its first key.)
    requests = [(703, 1), (700, 7 if hq == 8 else 2), (295, 40), (944, 12), (65, 3)]
    st = Step8(dev, requests, hq, 2, d, ps, window, sinks, seed=d + ps)
    for scale in SCALES:
        assert spoil(st, scale) > 20
        st.o.fill_(3.0)
        print(f"[fp8] hidden scale {scale}: {hq}/2 D={d} pages of {ps}, window {window} sinks {sinks}", flush=True)
        st.run()


@pytest.mark.parametrize("scale", [2.0 ** 120, 2.0 ** 127, float("nan"), 0.0])
@pytest.mark.parametrize("ps", [16, 32])
@pytest.mark.parametrize("d", [64, 128])
def test_entries_of_pages_behind_the_window(dev, d, ps, scale):
    """Pages that no row sees any more have no entry: 0xFFFFFFFF reads as the last
    page, which nobody has written."""
    requests = [(703, 1), (700, 7), (295, 40), (944, 12)]
    st = Step8(dev, requests, 8, 2, d, ps, 100, 20, seed=ps)
    last = torch.full((1, st.stride), 0x7E, dtype=torch.uint8, device=dev)
    n = st.hkv * ps * d
    last[:, n:n + st.hkv * ps // 4].view(torch.float32).fill_(scale)
    st.k, st.v = torch.cat([st.k, last]), torch.cat([st.v, last])
    st.pages += 1
    table, gone = st.table.cpu().numpy(), 0
    for b, (length, new) in enumerate(requests):
        low = length - new + 1 - 100
        for page in range(low // ps):
            if page * ps >= 20:
                table[b, page] = -1
                gone += 1
    assert gone > 20
    st.table.copy_(torch.from_numpy(np.ascontiguousarray(table)))
    st.run()
    print(f"[fp8] entries gone: D={d} pages of {ps}, scale {scale}: {shape_of(st)}", flush=True)


@pytest.mark.parametrize("d", [64, 128])
def test_hidden_blocks_in_pieces(dev, d):
    """A window as long as many tiles, whose unit is cut into pieces that meet in the
    merge."""
    st = Step8(dev, [(5003, 1), (4990, 6)], 8, 2, d, 16, 4000, 20, seed=d)
    st.make_plan()
    for scale in (2.0 ** 120, 3e38, float("inf")):
        assert spoil(st, scale) > 50
        st.o.fill_(3.0)
        st.run()
    assert shape_of(st)[1]
