"""The 8-bit paged cache restated in numpy: its format bit by bit, and what a
write does to the blocks that it touches."""
from __future__ import annotations

import numpy as np

BLOCK, LOW, HIGH, LARGEST = 16, -100, 119, 448.0


def _values():
    out = np.empty(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        x = float("nan") if c & 127 == 127 else m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[c] = -x if c & 128 else x
    return out


VALUES = _values()                       # of each code
_STEPS = VALUES[:127]                    # ascending, codes 0..126
_HALVES = (_STEPS[:-1] + _STEPS[1:]) / 2


def encode(x):
    """Nearest codes of float64 x, halves to even codes; past 448: 448, not
    finite: NaN, with the sign."""
    x = np.asarray(x, np.float64)
    size = np.minimum(np.abs(x), LARGEST)
    code = np.searchsorted(_HALVES, size, side="left")
    tie = (code < 126) & (size == _HALVES[np.minimum(code, 125)])
    code = np.where(tie & (code % 2 == 1), code + 1, code)
    code = np.where(np.isfinite(x), code, 127)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def exponent_for(most):
    """The least e in LOW..HIGH with most <= 448 * 2^e (HIGH if there is none)."""
    e = LOW
    while e < HIGH and most > LARGEST * 2.0 ** e:
        e += 1
    return e


def page_bytes(ps, hkv, d):
    return -(-(hkv * ps * d + hkv * ps // BLOCK * 4) // 16) * 16


class Cache:
    """A K or V cache: [pages][stride] bytes, all ones at first (codes and scales
    that are NaN)."""

    def __init__(self, pages, ps, hkv, d, stride=None):
        self.pages, self.ps, self.hkv, self.d = pages, ps, hkv, d
        self.raw = np.full((pages, stride or page_bytes(ps, hkv, d)), 255, np.uint8)

    def codes(self):
        n = self.hkv * self.ps * self.d
        return self.raw[:, :n].reshape(self.pages, self.hkv, self.ps, self.d)

    def put_codes(self, page, row, codes):
        n = self.ps * self.d
        for h in range(self.hkv):
            at = h * n + row * self.d
            self.raw[page, at:at + self.d] = codes[h]

    def _scale_span(self, page, h, block):
        at = self.hkv * self.ps * self.d + 4 * (h * (self.ps // BLOCK) + block)
        return self.raw[page, at:at + 4]

    def scale(self, page, h, block):
        return float(self._scale_span(page, h, block).copy().view(np.float32)[0])

    def put_scale(self, page, h, block, s):
        self._scale_span(page, h, block)[:] = np.array([s], np.float32).view(np.uint8)

    def row(self, slot):
        """[heads][dims] values in slot."""
        page, r = divmod(int(slot), self.ps)
        codes = self.codes()[page, :, r]
        s = np.array([self.scale(page, h, r // BLOCK) for h in range(self.hkv)])
        return VALUES[codes] * s[:, None]

    def write(self, slots, rows, exponents=None):
        """rows [T][heads][dims] float64 into slots; rows whose slot is past the
        cache are left out.  exponents {(block, head): e}: those, where they are
        known otherwise."""
        by_block = {}
        for t, s in enumerate(int(x) for x in slots):
            if s < self.pages * self.ps:
                by_block.setdefault(s // BLOCK, []).append(t)
        for block, ts in by_block.items():
            page, b = divmod(block, self.ps // BLOCK)
            new = {int(slots[t]) % BLOCK: t for t in ts}
            for h in range(self.hkv):
                old = self.scale(page, h, b)
                valid = old in POWERS
                x = np.abs(np.array([rows[t][h] for t in ts]))
                e = exponent_for(np.where(np.isfinite(x), x, 0.0).max())
                if valid and 0 not in new:
                    e = max(e, POWERS[old])
                if exponents is not None:
                    e = exponents[block, h]
                for r in range(BLOCK):
                    at = h * self.ps * self.d + (b * BLOCK + r) * self.d
                    span = self.raw[page, at:at + self.d]
                    if r in new:
                        span[:] = encode(rows[new[r]][h] * 2.0 ** -e)
                    elif valid and 0 not in new and 2.0 ** e != old:
                        span[:] = encode(VALUES[span] * old * 2.0 ** -e)
                self.put_scale(page, h, b, 2.0 ** e)


POWERS = {2.0 ** e: e for e in range(LOW, HIGH + 1)}
