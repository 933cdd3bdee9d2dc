"""The 8-bit paged cache without a GPU: argument checks of its entry points and
the oracle that the GPU tests use."""
import numpy as np
import pytest
import torch

from tests import fp8_oracle as F8
from tests.test_paged_host import G, INVALID, UNSUPPORTED, WORKSPACE, bad
from toyinfer_amd import attn

L = attn.LIB
PAGE = 16 * 8 * 128 + 8 * 4


@pytest.mark.parametrize("ps,hkv,d", [(16, 1, 64), (16, 8, 128), (64, 3, 64), (65536, 2, 128)])
def test_page_bytes(ps, hkv, d):
    n = attn.paged_fp8_page_bytes(ps, hkv, d)
    assert n == F8.page_bytes(ps, hkv, d) and n % 16 == 0
    assert 0 <= n - (hkv * ps * d + hkv * ps // 16 * 4) < 16


@pytest.mark.parametrize("ps,hkv,d", [(8, 8, 128), (24, 8, 128), (0, 8, 128), (1 << 17, 8, 128),
                                      (16, 0, 128), (16, 8, 96)])
def test_page_bytes_of_other_sizes(ps, hkv, d):
    assert attn.paged_fp8_page_bytes(ps, hkv, d) == 0
    with pytest.raises(attn.ToyInferError):
        attn.paged_fp8_cache(2, ps, hkv, d, "cpu")


def test_prologue_validation():
    fn = L.toyinfer_paged_qkv_prologue_fp8
    #       q  k      v      qw     kw     rope   npos pos   slot   t  eps   q_out  kc     vc      pages ps stride hq hkv d
    args = [G, 2 * G, 3 * G, 4 * G, 5 * G, 6 * G, 99, 7 * G, 8 * G, 5, 1e-6, 9 * G, 10 * G, 11 * G, 7, 16,
            PAGE, 16, 8, 128, None]
    for i in (0, 1, 2, 3, 4, 5, 7, 8, 11, 12, 13):
        bad(fn, args, i, None, INVALID)
        bad(fn, args, i, args[i] + 2, INVALID)
    for i in (6, 9, 14, 17, 18):
        bad(fn, args, i, 0, INVALID)
    for ps in (0, 8, 17, 1 << 17):
        bad(fn, args, 15, ps, INVALID)
    bad(fn, args, 16, PAGE - 16, INVALID)         # pages on each other
    bad(fn, args, 16, PAGE + 8, INVALID)          # rows off 16 bytes
    bad(fn, args, 16, 1 << 41, UNSUPPORTED)
    bad(fn, args, 18, 3, INVALID)                 # 16 % 3
    bad(fn, args, 19, 96, UNSUPPORTED)
    bad(fn, args, 14, 1 << 28, UNSUPPORTED)       # slots past 32 bits
    bad(fn, args, 9, 1 << 27, UNSUPPORTED)
    bad(fn, args, 13, 10 * G, INVALID)            # one cache for both
    bad(fn, args, 13, 10 * G + PAGE // 2 // 16 * 16, INVALID)  # V's pages in the middle of K's
    bad(fn, args, 11, G + 32, INVALID)            # q_out across q
    bad(fn, args, 11, 2 * G, INVALID)             # q_out over k
    bad(fn, args, 12, G, INVALID)                 # K cache over q
    bad(fn, args, 13, 9 * G, INVALID)             # V cache over q_out


def test_span_limit():
    """Caches past what 47 bits address are refused before a product can wrap."""
    fn = L.toyinfer_paged_qkv_prologue_fp8
    args = [G, 2 * G, 3 * G, 4 * G, 5 * G, 6 * G, 99, 7 * G, 8 * G, 5, 1e-6, 9 * G, 10 * G, 11 * G, (1 << 24) + 1,
            16, 1 << 24, 16, 8, 128, None]
    assert fn(*args) == UNSUPPORTED


def test_read_validation():
    fn = L.toyinfer_paged_kv_read_fp8
    #       kc vc     table  start  lens   b  rows ko    vo     pages ps stride blocks hkv d
    args = [G, 2 * G, 3 * G, 4 * G, 5 * G, 4, 33, 6 * G, 7 * G, 9, 16, PAGE, 8, 8, 128, None]
    for i in (0, 1, 2, 3, 4, 7, 8):
        bad(fn, args, i, None, INVALID)
        bad(fn, args, i, args[i] + 2, INVALID)
    for i in (5, 6, 9, 12, 13):
        bad(fn, args, i, 0, INVALID)
    for ps in (8, 48):
        bad(fn, args, 10, ps, INVALID)
    bad(fn, args, 11, PAGE - 16, INVALID)
    bad(fn, args, 14, 80, UNSUPPORTED)
    bad(fn, args, 5, 4097, UNSUPPORTED)
    bad(fn, args, 12, 1 << 27, UNSUPPORTED)
    bad(fn, args, 8, 6 * G + 16, INVALID)         # the outputs on each other
    bad(fn, args, 7, G + 64, INVALID)             # rows over the cache
    bad(fn, args, 8, 4 * G, INVALID)              # rows over query_start


def test_attention_validation():
    plan_bytes = attn.paged_attention_plan_bytes(4, 33, 16, 8, 128)
    ws_bytes = attn.paged_attention_workspace_bytes(16, 8, 128)
    fn = L.toyinfer_paged_attention_fp8
    #       q  kc     vc     o      table  plan   bytes       b  rows pages ps stride blocks w s hq hkv d
    args = [G, 2 * G, 3 * G, 4 * G, 5 * G, 6 * G, plan_bytes, 4, 33, 9, 16, PAGE, 8, 0, 0, 16, 8, 128,
            7 * G, ws_bytes, None]
    for i in (0, 1, 2, 3, 4, 5, 18):
        bad(fn, args, i, None, INVALID)
        bad(fn, args, i, args[i] + 2, INVALID)
    for i in (7, 8, 9, 12, 15, 16):
        bad(fn, args, i, 0, INVALID)
    for ps in (8, 48):
        bad(fn, args, 10, ps, INVALID)
    bad(fn, args, 11, PAGE - 16, INVALID)
    bad(fn, args, 17, 80, UNSUPPORTED)
    bad(fn, args, 6, plan_bytes - 256, WORKSPACE)
    bad(fn, args, 19, ws_bytes - 1, WORKSPACE)
    bad(fn, args, 3, G, INVALID)              # o over q
    bad(fn, args, 3, 2 * G + 16, INVALID)     # o over the cache
    bad(fn, args, 18, 6 * G, INVALID)         # workspace over the plan


@pytest.mark.parametrize("view,stride,ok", [
    (lambda t: t, 1, True),
    (lambda t: t[1:], 1, True),
    (lambda t: t.view(3, 2, PAGE)[:, 0], 2, True),       # beside V's pages
    (lambda t: t.view(3, 2, PAGE)[:, 1], 2, True),
    (lambda t: t.view(3, 2, PAGE)[:, 0], 1, False),
    (lambda t: t.view(torch.int8), 1, False),
    (lambda t: t.view(-1), 1, False),
    (lambda t: t[:, 16:], 1, False),                     # less than a page
    (lambda t: t[:1], 1, False),                         # fewer pages
    (lambda t: t.t().contiguous().t(), 1, False),
])
def test_binding_takes_caches_of_pages_only(view, stride, ok):
    t = view(torch.zeros(6, PAGE, dtype=torch.uint8))
    args = "paged", -1, 2, 16, stride * PAGE, 8, 128
    if ok:
        attn._need_cache_fp8(*args, t)
    else:
        with pytest.raises(attn.ToyInferError):
            attn._need_cache_fp8(*args, t)


def test_binding_takes_device_tensors_only():
    i = torch.zeros(64, dtype=torch.int32)
    b = torch.zeros(4096, dtype=torch.bfloat16)
    c = attn.paged_fp8_cache(1, 16, 1, 128, "cpu")
    n = c.shape[1]
    for call in (lambda: attn.paged_qkv_prologue_fp8(b, b, b, b, b, b.float(), 2, i, i, 1, 1e-6, b, c, c, 1,
                                                     16, n, 1, 1, 128),
                 lambda: attn.paged_kv_read_fp8(c, c, i, i, i, 1, 1, b, b, 1, 16, n, 1, 1, 128),
                 lambda: attn.paged_attention_fp8(b, c, c, b, i, i, 1, 1, 1, 16, n, 1, 0, 0, 1, 1, 128, i)):
        with pytest.raises(attn.ToyInferError) as e:
            call()
        assert e.value.status == INVALID


# ------------------------------------------------------------------ oracle

def test_oracle_codes():
    """Every code is its own value's, halves go to even codes, and torch's
    conversion to the type agrees on values that it holds."""
    finite = np.array([c for c in range(256) if c & 127 != 127])
    assert (F8.encode(F8.VALUES[finite]) == finite).all()
    assert F8.VALUES[126] == 448 and F8.VALUES[1] == 2.0 ** -9 and F8.VALUES[8] == 2.0 ** -6
    assert F8.encode([1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 460.0, 1e9]).tolist() == [56, 58, 0, 2, 126, 126]
    assert F8.encode([float("nan"), float("inf"), -float("inf"), -0.0]).tolist() == [127, 127, 255, 128]
    x = np.random.default_rng(0).standard_normal(20000) * np.exp2(np.random.default_rng(1).integers(-12, 8, 20000))
    x = np.clip(x, -448, 448).astype(np.float32)
    t = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert (F8.encode(x) == t).all()


def test_oracle_rounding_is_half_a_step():
    x = np.random.default_rng(2).standard_normal(10000) * 50
    off = np.abs(F8.VALUES[F8.encode(x)] - np.clip(x, -448, 448))
    assert (off <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10)).all()


@pytest.mark.parametrize("most,e", [(448.0, 0), (448.1, 1), (224.0, -1), (1.75, -8), (1.76, -7), (0.0, -100),
                                    (1e-35, -100), (3.0e38, 119), (1.75 * 2.0 ** 127, 119)])
def test_oracle_exponents(most, e):
    assert F8.exponent_for(most) == e


def test_oracle_write():
    """A block opens, grows, keeps its scale, and opens again."""
    c = F8.Cache(2, 16, 1, 64)
    row = lambda x: np.full((1, 64), x)
    c.write([16, 17], [row(1.0), row(0.5)])
    assert c.scale(1, 0, 0) == 2.0 ** -8 and (c.row(16) == 1).all() and np.isnan(c.row(18)).all()
    c.write([18], [row(100.0)])
    assert c.scale(1, 0, 0) == 2.0 ** -2 and (c.row(16) == 1).all() and (c.row(18) == 96).all()
    c.write([19], [row(3.0)])
    assert c.scale(1, 0, 0) == 2.0 ** -2 and (c.row(17) == 0.5).all() and (c.row(19) == 3).all()
    c.write([16, 99, 0xFFFFFFFF], [row(2.0)] * 3)
    assert c.scale(1, 0, 0) == 2.0 ** -7 and np.isnan(c.row(0)).all()
