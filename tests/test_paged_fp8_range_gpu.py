"""Keys at the ends of bf16's range on their way into the 8-bit paged cache: what the
norm's definition gives is small and finite, and gets the nearest code, however
large or small a value's product with its weight is before the norm divides."""
import numpy as np
import pytest
import torch

from tests import helpers as H
from tests import paged_oracle as PO
from tests.test_paged_fp8_gpu import POSITIONS, Writer, bf16
from tests.test_paged_gpu import ints
from toyinfer_amd import attn

pytestmark = pytest.mark.gpu

LARGEST = float(torch.finfo(torch.bfloat16).max)


def check_keys(dev, d, size, weight, eps):
    """Bit for bit the codes and scales of the values in 64 bits, as for ordinary keys;
    in every third row one value is bf16's largest."""
    w = Writer(dev, 9, 16, 2, 2, d, seed=d)
    w.kw = bf16(w.rng.uniform(0.5, 1.5, d) * weight)
    t = 100
    x = np.clip(w.rng.standard_normal((t, 2, d)) * size, -LARGEST, LARGEST)
    x[::3, :, 5] = LARGEST * (1 - 2 * (np.arange(-(-t // 3)) % 2))[:, None]
    k, v, q = bf16(x), w.rows(t), bf16(w.rng.standard_normal((t, 2, d)))
    slots, pos = np.arange(t) + 16, np.arange(t) % POSITIONS
    q_out = torch.empty_like(q, device=dev)
    print(f"[fp8] keys of {size} by {weight}, D={d} eps {eps}", flush=True)
    attn.paged_qkv_prologue_fp8(q.to(dev), k.to(dev), v.to(dev), w.qw.to(dev), w.kw.to(dev), w.rope.to(dev), POSITIONS,
                                ints(pos, dev), ints(slots, dev), t, eps, q_out, w.k_d, w.v_d, w.pages, w.ps,
                                w.k_d.stride(0), 2, 2, d)
    H.sync()
    y = PO.rms_rope(k.double().numpy(), w.kw.double().numpy(), w.rope.double().numpy()[pos], float(np.float32(eps)))
    assert np.isfinite(y).all()
    w.k.write(slots, y)
    w.v.write(slots, v.double().numpy())
    got = w.k_d.cpu().numpy()
    assert (got == w.k.raw).all(), f"{int((got != w.k.raw).sum())} bytes"
    assert (w.v_d.cpu().numpy() == w.v.raw).all()
    return y


@pytest.mark.parametrize("eps", [1e-6, 0.0])
@pytest.mark.parametrize("size,weight", [
    (2.0 ** 125, 2.0 ** 10),    # products past the largest fp32
    (2.0 ** 125, 2.0 ** 115),
    (2.0 ** 20, 2.0 ** 120),
    (2.0 ** 125, 2.0 ** -90),
    (2.0 ** -100, 2.0 ** -30),  # below the normal ones, and below all
    (2.0 ** -120, 2.0 ** -60),
    (2.0 ** -130, 1.0),         # subnormal themselves
    (1.0, 1.0),
])
@pytest.mark.parametrize("d", [64, 128])
def test_keys_get_the_nearest_code(dev, d, size, weight, eps):
    check_keys(dev, d, size, weight, eps)


@pytest.mark.parametrize("d", [64, 128])
def test_keys_past_the_largest_fp32(dev, d):
    """Finite keys that fp32 does not hold take the largest code under the largest scale."""
    y = check_keys(dev, d, 1.0, 2.0 ** 127, 1e-6)
    assert (np.abs(y) > float(np.finfo(np.float32).max)).sum() > 100
