"""Limits of the paged cache's size, at the C ABI, without a GPU."""
import pytest

from toyinfer_amd import attn

G = 1 << 50  # stand-in addresses; never dereferenced here


@pytest.mark.parametrize("pages,stride,status", [
    (1 << 27, 1 << 39, attn.ERR_UNSUPPORTED),       # the span passes 64 bits of bytes
    (1 << 20, 1 << 27, attn.ERR_UNSUPPORTED),       # 2^47 elements
    (3, 1 << 40, attn.ERR_UNSUPPORTED),
    (0xFFFFFFFF, 1 << 14, attn.ERR_UNSUPPORTED),    # slots past 32 bits
])
def test_caches_beyond_any_memory(pages, stride, status):
    """A span that wraps must not pass the checks for overlap."""
    prologue = attn.LIB.toyinfer_paged_qkv_prologue_bf16(
        G, 2 * G, 3 * G, 4 * G, 5 * G, 6 * G, 99, 7 * G, 8 * G, 5, 1e-6, 9 * G, 10 * G, 11 * G, pages,
        16, stride, 16, 8, 128, None)
    attention = attn.LIB.toyinfer_paged_attention_bf16(
        G, 2 * G, 3 * G, 4 * G, 5 * G, 6 * G, 1 << 40, 4, 33, pages, 16, stride, 8, 0, 0, 16, 8, 128,
        7 * G, 1 << 40, None)
    assert (prologue, attention) == (status, status)
