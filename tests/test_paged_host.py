"""Argument checks of the paged-cache entry points, without a GPU."""
import numpy as np
import pytest
import torch

from tests import paged_oracle as PO
from toyinfer_amd import attn

L = attn.LIB
INVALID, UNSUPPORTED, WORKSPACE = (attn.ERR_INVALID_ARGUMENT, attn.ERR_UNSUPPORTED,
                                   attn.ERR_WORKSPACE)
G = 1 << 40  # stand-in addresses this far apart; never dereferenced here


def bad(fn, args, at, value, status):
    a = list(args)
    a[at] = value
    assert fn(*a) == status, (fn.__name__, at, value)


def test_tables_validation():
    fn = L.toyinfer_paged_tables_u32
    #       ctx new  batch free cap num_free ps table blocks rows qs     sl      pos     slot    status
    args = [G, 2 * G, 4, 3 * G, 9, 4 * G, 16, 5 * G, 8, 32, 6 * G, 7 * G, 8 * G, 9 * G, 10 * G, None]
    for i in (0, 1, 3, 5, 7, 10, 11, 12, 13, 14):
        bad(fn, args, i, None, INVALID)
        bad(fn, args, i, args[i] + 2, INVALID)
    for i in (2, 8, 9):
        bad(fn, args, i, 0, INVALID)
    for ps in (0, 4, 12, 24, 1 << 17):
        bad(fn, args, 6, ps, INVALID)
    bad(fn, args, 2, 4097, UNSUPPORTED)
    bad(fn, args, 8, 1 << 27, UNSUPPORTED)      # positions past 2^31
    bad(fn, args, 9, 1 << 31, UNSUPPORTED)
    bad(fn, args, 11, G, INVALID)               # seq_lens over context_lens
    bad(fn, args, 14, 4 * G, INVALID)           # status over num_free
    bad(fn, args, 12, 9 * G + 4, INVALID)       # two outputs on each other
    bad(fn, args, 10, 5 * G + 4 * 31, INVALID)  # query_start in the tables' last entry


def test_prologue_validation():
    fn = L.toyinfer_paged_qkv_prologue_bf16
    #       q  k      v      qw     kw     rope   npos pos   slot   t  eps   q_out  kc     vc      pages ps stride hq hkv d
    args = [G, 2 * G, 3 * G, 4 * G, 5 * G, 6 * G, 99, 7 * G, 8 * G, 5, 1e-6, 9 * G, 10 * G, 11 * G, 7, 16,
            16 * 8 * 128, 16, 8, 128, None]
    for i in (0, 1, 2, 3, 4, 5, 7, 8, 11, 12, 13):
        bad(fn, args, i, None, INVALID)
        bad(fn, args, i, args[i] + 2, INVALID)
    for i in (6, 9, 14, 17, 18):
        bad(fn, args, i, 0, INVALID)
    for ps in (0, 4, 17):
        bad(fn, args, 15, ps, INVALID)
    bad(fn, args, 16, 16 * 8 * 128 - 8, INVALID)  # pages on each other
    bad(fn, args, 16, 16 * 8 * 128 + 4, INVALID)  # rows off 16 bytes
    bad(fn, args, 18, 3, INVALID)                 # 16 % 3
    bad(fn, args, 19, 96, UNSUPPORTED)
    bad(fn, args, 14, 1 << 28, UNSUPPORTED)       # slots past 32 bits
    bad(fn, args, 9, 1 << 27, UNSUPPORTED)
    bad(fn, args, 13, 10 * G, INVALID)            # one cache for both
    bad(fn, args, 13, 10 * G + 16 * 8 * 128, INVALID)  # V's pages in the middle of K's
    bad(fn, args, 11, G + 32, INVALID)            # q_out across q
    bad(fn, args, 11, 2 * G, INVALID)             # q_out over k
    bad(fn, args, 12, G, INVALID)                 # K cache over q
    bad(fn, args, 13, 9 * G, INVALID)             # V cache over q_out


def test_attention_validation():
    plan_bytes = attn.paged_attention_plan_bytes(4, 33, 16, 8, 128)
    ws_bytes = attn.paged_attention_workspace_bytes(16, 8, 128)
    assert plan_bytes > 0 and ws_bytes > 0
    assert attn.paged_attention_plan_bytes(0, 33, 16, 8, 128) == 0
    assert attn.paged_attention_plan_bytes(4, 33, 16, 7, 128) == 0
    assert attn.paged_attention_workspace_bytes(16, 8, 96) == 0
    # Units: one per request and 32 rows at most, whatever the cut.
    assert attn.paged_attention_plan_bytes(4, 1 << 20, 32, 8, 128) > (1 << 20) * 4 // 32 * 48

    fn = L.toyinfer_paged_attention_plan
    #       qs  lens  b  rows ps  blocks w s hq hkv d  plan
    args = [G, 2 * G, 4, 33, 16, 8, 0, 0, 16, 8, 128, 3 * G, plan_bytes, None]
    for i in (0, 1, 11):
        bad(fn, args, i, None, INVALID)
    bad(fn, args, 0, G + 1, INVALID)
    bad(fn, args, 11, 3 * G + 128, INVALID)
    for i in (2, 3, 5, 8, 9):
        bad(fn, args, i, 0, INVALID)
    bad(fn, args, 4, 20, INVALID)
    bad(fn, args, 2, 4097, UNSUPPORTED)
    bad(fn, args, 3, 1 << 30, UNSUPPORTED)
    bad(fn, args, 5, 1 << 27, UNSUPPORTED)
    bad(fn, args, 10, 256, UNSUPPORTED)
    bad(fn, args, 12, plan_bytes - 1, WORKSPACE)
    bad(fn, args, 0, 3 * G + 64, INVALID)  # lengths inside the plan

    fn = L.toyinfer_paged_attention_bf16
    #       q  kc     vc     o      table  plan   bytes       b  rows pages ps stride        blocks w s hq hkv d
    args = [G, 2 * G, 3 * G, 4 * G, 5 * G, 6 * G, plan_bytes, 4, 33, 9, 16, 16 * 8 * 128, 8, 0, 0, 16, 8, 128,
            7 * G, ws_bytes, None]
    for i in (0, 1, 2, 3, 4, 5, 18):
        bad(fn, args, i, None, INVALID)
        bad(fn, args, i, args[i] + 2, INVALID)
    for i in (7, 8, 9, 12, 15, 16):
        bad(fn, args, i, 0, INVALID)
    bad(fn, args, 10, 48, INVALID)
    bad(fn, args, 11, 16 * 8 * 128 - 8, INVALID)
    bad(fn, args, 17, 80, UNSUPPORTED)
    bad(fn, args, 6, plan_bytes - 256, WORKSPACE)
    bad(fn, args, 19, ws_bytes - 1, WORKSPACE)
    bad(fn, args, 3, G, INVALID)              # o over q
    bad(fn, args, 3, 2 * G + 16, INVALID)     # o over the cache
    bad(fn, args, 18, 6 * G, INVALID)         # workspace over the plan


def test_binding_takes_dense_device_tensors_only():
    """Host tensors, other types and strided views are refused by the binding
    before any address is passed on."""
    i = torch.zeros(64, dtype=torch.int32)
    with pytest.raises(attn.ToyInferError) as e:
        attn.paged_tables_u32(i, i, 4, i, 8, i, 16, i, 8, 32, i, i, i, i, i)
    assert e.value.status == INVALID
    b = torch.zeros(4096, dtype=torch.bfloat16)
    with pytest.raises(attn.ToyInferError):
        attn.paged_qkv_prologue_bf16(b, b, b, b, b, b.float(), 2, i, i, 1, 1e-6, b, b, b, 1, 8, 1024, 1, 1, 128)
    with pytest.raises(attn.ToyInferError):
        attn.paged_attention_plan(i, i, 4, 33, 16, 8, 0, 0, 16, 8, 128, i)
    with pytest.raises(attn.ToyInferError):
        attn.paged_attention_bf16(b, b, b, b, i, i, 1, 1, 1, 8, 1024, 1, 0, 0, 1, 1, 128, i)


def test_oracle_of_the_tables():
    """The plain form itself, on a step small enough to read."""
    table = np.full((3, 3), 9, np.uint32)
    start, seq, pos, slot, table, status = PO.tables([3, 8, 0], [6, 1, 0], [5, 6, 7], 8, table, 9)
    assert start == [0, 6, 7, 7] and seq == [9, 9, 0] and status == [1, 0]
    assert pos == [3, 4, 5, 6, 7, 8, 8, 0, 0]
    assert table.tolist() == [[9, 7, 9], [9, 6, 9], [9, 9, 9]]
    assert slot == [75, 76, 77, 78, 79, 56, 48, PO.NO_SLOT, PO.NO_SLOT]


def test_oracle_of_the_attention_mask():
    seen = PO.visible(2, 6, 2, 1)
    assert seen.astype(int).tolist() == [[1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    o, away, size = PO.attention(torch.zeros(1, 1, 1), torch.zeros(2, 1, 1),
                                 torch.tensor([[[1.0]], [[3.0]]]), 0, 0)
    assert o.item() == 2 and away.item() == 1 and size.item() == 2


@pytest.mark.parametrize("view,stride,ok", [
    (lambda t: t, 1, True),
    (lambda t: t.view(-1), 1, True),
    (lambda t: t.view(48, 2, 64), 1, True),
    (lambda t: t[1:], 1, True),
    (lambda t: t.view(3, 2, 8, 2, 64)[:, 0], 2, True),           # beside V's pages
    (lambda t: t.view(3, 2, 8, 2, 64)[:, 1:], 2, True),
    (lambda t: t.view(3, 2, 8, 2, 64), 2, True),
    (lambda t: t.view(-1)[:2 * 8 * 2 * 64], 1, True),
    (lambda t: t.view(3, 2, 8, 2, 64)[:, 0], 1, False),          # pages closer than they lie
    (lambda t: t, 2, False),                                     # further apart
    (lambda t: t.view(6, 2, 8, 64), 1, False),                   # [heads][rows]
    (lambda t: t.view(6, 2, 8, 64).transpose(1, 2), 1, False),
    (lambda t: t.view(6, 8, 64, 2).transpose(2, 3), 1, False),
    (lambda t: t.view(6, 8, 4, 32)[:, :, :2], 1, False),         # heads of a wider cache
    (lambda t: t.view(8, 6, 2, 64).transpose(0, 1), 1, False),   # pages inside rows
    (lambda t: t.view(48, 2, 64)[::2], 1, False),
])
def test_binding_takes_caches_of_pages_only(view, stride, ok):
    """A cache of another layout than the kernels read is refused, one in pages
    at the stride that is given taken."""
    t = view(torch.zeros(6, 8, 2, 64, dtype=torch.bfloat16))
    args = "paged", -1, 2, 8, stride * 8 * 2 * 64, 2, 64
    if ok:
        attn._need_cache(*args, t)
    else:
        with pytest.raises(attn.ToyInferError):
            attn._need_cache(*args, t)


def test_binding_takes_one_page_and_one_head():
    """Sizes of one have no stride that counts."""
    one = torch.zeros(1, 8, 2, 64, dtype=torch.bfloat16)
    attn._need_cache("paged", -1, 1, 8, 5000, 2, 64, one, one.view(-1))
    wide = torch.zeros(3, 8, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(attn.ToyInferError):
        attn._need_cache("paged", -1, 2, 8, 8 * 4 * 64, 1, 64, wide[:, :, 1:2])
    head = torch.zeros(3, 8, 64, dtype=torch.bfloat16)[:, :, None]
    attn._need_cache("paged", -1, 3, 8, 8 * 64, 1, 64, head)
    attn._need_cache("paged", -1, 1, 8, 8 * 2 * 64, 2, 64, one.view(1, 8, 128))  # heads and dims in one
