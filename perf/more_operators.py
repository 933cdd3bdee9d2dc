"""Performance cases of the paged cache in 8 bits: serving many requests at once
from half the cache.

A layer's K and V cache are pages of e4m3 codes with a scale, a power of two, for
each block of 16 tokens and KV head: a page is its codes [heads][rows][dims], then
its scales [heads][rows / 16] in fp32.  `write` normalises and rotates the new
tokens' Q and K, quantises K and V into their slots, and reads back every block
that this touched; `read` expands whole contexts to bf16; `attention` runs the new
tokens over the pages.  With `own` false `run` computes the same in elementary
torch operations; `exact` gives the results in 64 bits.

A block whose first row a call writes starts anew: its scale is the smallest 2^e
(e from -100 to 119) with which the largest written value is at most 448 * 2^e.
Otherwise its scale is the larger of that and the one it has, and where that makes
it grow, the rows that it keeps are rounded again.
"""
import math

import torch

own = False

EPS, THETA, POSITIONS = 1e-6, 1e6, 40960
BLOCK, LARGEST, LOW, HIGH = 16, 448.0, -100, 119
NO_SLOT = -1  # 0xFFFFFFFF as the int32 that torch holds


def listed():
    return [
        # A decode step of eight requests, Qwen3-0.6B heads: launch-bound.
        {"name": "write_decode_b8", "kind": "write", "mix": "decode", "b": 8, "new": 1,
         "ctx": 4096, "ps": 16, "hq": 16, "hkv": 8, "d": 128},
        # A second chat turn that begins inside a block.
        {"name": "write_chunk_t1371", "kind": "write", "mix": "chunk", "b": 1, "new": 1371,
         "ctx": 37, "ps": 16, "hq": 16, "hkv": 8, "d": 128},
        # Prompts of about 8192 tokens in all, Qwen3-8B heads.
        {"name": "write_chunk_b4", "kind": "write", "mix": "chunk", "b": 4, "new": 2500,
         "ctx": 512, "ps": 64, "hq": 32, "hkv": 8, "d": 128},
        # One chat's context expanded for a path that takes bf16.
        {"name": "read_b1_l1371", "kind": "read", "mix": "decode", "b": 1, "new": 1,
         "ctx": 1371, "ps": 16, "hq": 16, "hkv": 8, "d": 128},
        # Long conversations expanded together.
        {"name": "read_b16_l8192", "kind": "read", "mix": "decode", "b": 16, "new": 1,
         "ctx": 8192, "ps": 64, "hq": 32, "hkv": 8, "d": 128},
        # The next token of one chat: latency.
        {"name": "decode_b1_l1371", "kind": "attention", "mix": "decode", "b": 1, "new": 1,
         "ctx": 1371, "ps": 16, "window": 0, "sinks": 0, "hq": 16, "hkv": 8, "d": 128},
        # The next token of 48 requests of different lengths.
        {"name": "decode_b48_l8192", "kind": "attention", "mix": "decode", "b": 48, "new": 1,
         "ctx": 8192, "ps": 16, "window": 0, "sinks": 0, "hq": 32, "hkv": 8, "d": 128},
        # The same at head_dim 64, deep in long conversations under a window with sinks.
        {"name": "decode_b32_window_d64", "kind": "attention", "mix": "decode", "b": 32, "new": 1,
         "ctx": 32768, "ps": 64, "window": 4096, "sinks": 4, "hq": 32, "hkv": 8, "d": 64},
        # The next piece of one long prompt.
        {"name": "chunk_t512_l8192", "kind": "attention", "mix": "chunk", "b": 1, "new": 512,
         "ctx": 7680, "ps": 16, "window": 0, "sinks": 0, "hq": 32, "hkv": 8, "d": 128},
        # Decoding requests and a few prompt pieces in one batch, an odd group of heads.
        {"name": "mixed_b24_g3", "kind": "attention", "mix": "mixed", "b": 24, "new": 777,
         "ctx": 5000, "ps": 32, "window": 0, "sinks": 0, "hq": 24, "hkv": 8, "d": 128},
        # A whole long prompt into empty pages.
        {"name": "prompt_t8192", "kind": "attention", "mix": "chunk", "b": 1, "new": 8192,
         "ctx": 0, "ps": 16, "window": 0, "sinks": 0, "hq": 32, "hkv": 8, "d": 128},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attention", "attention", "attention"])
    hq, hkv = rng.choice([(16, 8), (32, 8), (8, 8), (12, 2), (6, 2), (5, 1), (24, 8), (28, 4)])
    c = {"kind": kind, "ps": rng.choice([16, 16, 32, 64, 128, 256]), "hq": hq, "hkv": hkv,
         "d": rng.choice([128, 128, 64])}
    if kind == "write":
        c["mix"] = rng.choice(["decode", "chunk", "mixed"])
        c["b"] = _log_int(rng, 1, 256)
        c["new"] = (rng.randint(1, 4) if c["mix"] == "decode"
                    else _log_int(rng, 2, 8192 // c["b"] + 2))
        c["ctx"] = _log_int(rng, 1, 8192)
        return c
    if kind == "read":
        c["mix"], c["new"] = "decode", 1
        c["b"] = _log_int(rng, 1, 64)
        c["ctx"] = _log_int(rng, 1, (1 << 17) // c["b"])
        return c
    # At most the longest listed prompt's products (new tokens times context)
    # and the longest listed batch's cache.
    c["mix"] = rng.choice(["decode", "chunk", "mixed"])
    c["b"] = _log_int(rng, 1, 64 if c["mix"] == "decode" else 24)
    c["new"] = (rng.randint(1, 4) if c["mix"] == "decode"
                else _log_int(rng, 2, 4096 // c["b"] + 2))
    c["ctx"] = _log_int(rng, 1, min(32768, (1 << 24) // (c["b"] * c["new"]), (1 << 18) // c["b"]))
    c["window"] = rng.choice([0, 0, _log_int(rng, 1, 4096)])
    c["sinks"] = rng.choice([0, 1, 4, 37]) if c["window"] else 0
    return c


# ------------------------------------------------------------------ inputs

def _lengths(case, seed):
    """(cached, new) per request.  Decode: every request `new` tokens; chunk:
    every request `new` or down to half as many; mixed: one request in eight a
    chunk, one in sixteen idle, the others one token; all have a quarter of `ctx`
    cached or up to all of it.  The seed orders them."""
    b, new, ctx = case["b"], case["new"], case["ctx"]
    u = torch.rand(b, generator=torch.Generator().manual_seed(b)).tolist()
    cached = [ctx - int(0.75 * ctx * x) if i else ctx for i, x in enumerate(u)]
    fresh = []
    for i in range(b):
        if case["mix"] == "decode":
            fresh.append(new)
        elif case["mix"] == "chunk" or i % 8 == 0:
            fresh.append(new - new // 2 * i // b)
        else:
            fresh.append(0 if i % 16 == 9 else 1)
    order = torch.randperm(b, generator=torch.Generator().manual_seed(seed)).tolist()
    return [cached[i] for i in order], [fresh[i] for i in order]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(n):
    s = [0]
    for x in n:
        s.append(s[-1] + x)
    return s


def _rope(d):
    inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    ang = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float()


def _page_bytes(case):
    rows = case["hkv"] * case["ps"]
    return -(-(rows * case["d"] + rows // BLOCK * 4) // 16) * 16


def _codes(cache, case):
    """[pages][heads][rows][dims] as they lie in the pages, uint8."""
    hkv, ps, d = case["hkv"], case["ps"], case["d"]
    return cache[:, :hkv * ps * d].view(-1, hkv, ps, d)


def _scales(cache, case):
    """[pages][heads][blocks], fp32."""
    hkv, ps, d = case["hkv"], case["ps"], case["d"]
    n = hkv * ps * d
    return cache[:, n:n + hkv * ps // BLOCK * 4].view(torch.float32).view(-1, hkv, ps // BLOCK)


def _filled(case, pages, g):
    """A cache whose pages all hold values, heads of different sizes."""
    hkv, ps, d = case["hkv"], case["ps"], case["d"]
    cache = torch.zeros(pages, _page_bytes(case), dtype=torch.uint8, device="cuda")
    size = torch.exp2(torch.rand(hkv, generator=g, device="cuda") * 3 - 2)[None, :, None, None]
    for i in range(0, pages, 1 + (1 << 26) // (hkv * ps * d)):
        part = cache[i:i + 1 + (1 << 26) // (hkv * ps * d)]
        x = torch.randn(part.shape[0], hkv, ps // BLOCK, BLOCK * d, generator=g, device="cuda") * size
        _, e = torch.frexp(x.abs().amax(-1) * (128 / LARGEST))
        scale = torch.ldexp(torch.ones_like(x[..., 0]), e - 7)
        _scales(part, case).copy_(scale)
        codes = (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        _codes(part, case).copy_(codes.view(-1, hkv, ps, d))
    return cache


def _inputs(case, seed):
    """What a case reads and the buffers it writes, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = torch.Generator().manual_seed(seed)
    kind, hq, hkv, d, ps = (case[k] for k in ("kind", "hq", "hkv", "d", "ps"))

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)

    cached, fresh = _lengths(case, seed)
    total = sum(fresh)
    lens = [c + n for c, n in zip(cached, fresh)]
    used = [-(-x // ps) for x in lens]
    blocks = max(used) + 1
    pages = sum(used) + 7
    order = torch.randperm(pages, generator=r).to(torch.int32)
    tables = torch.full((case["b"], blocks), NO_SLOT, dtype=torch.int32)
    for i, s in enumerate(_starts(used)[:-1]):
        tables[i, :used[i]] = order[s:s + used[i]]
    st = {"case": case, "lens": lens, "fresh": fresh, "total": total, "blocks": blocks,
          "pages": pages, "tables": tables.cuda(), "seq_lens": _ints(lens),
          "query_start": _ints(_starts(fresh)), "k_cache": _filled(case, pages, g),
          "v_cache": _filled(case, pages, g)}
    if kind == "attention":
        st.update(q=normal(total, hq, d, std=1.5),
                  o=torch.empty(total, hq, d, dtype=torch.bfloat16, device="cuda"))
        return st

    def slots_of(b, first, last):
        i = torch.arange(first, last)
        return tables[b][i // ps].long() * ps + i % ps

    # Of a read, whole contexts; of a write, the blocks that it touches.
    back = [x if kind == "read" else n + (x - n) % BLOCK if n else 0 for x, n in zip(lens, fresh)]
    st.update(back=sum(back), back_start=_ints(_starts(back)),
              back_slots=torch.cat([slots_of(b, x - m, x)
                                    for b, (x, m) in enumerate(zip(lens, back))]).cuda())
    for name in ("k_out", "v_out"):
        st[name] = torch.empty(sum(back), hkv, d, dtype=torch.bfloat16, device="cuda")
    if kind == "read":
        return st
    # A mixed step has rows for tokens that it does not fill.
    rows = total + total // 10 if case["mix"] == "mixed" else total
    slots = torch.cat([slots_of(b, x - n, x) for b, (x, n) in enumerate(zip(lens, fresh))])
    positions = torch.cat([torch.arange(x - n, x) for x, n in zip(lens, fresh)])
    st.update(rows=rows, q=normal(rows, hq, d, std=2.0),
              k=normal(rows, hkv, d, std=2.0), v=normal(rows, hkv, d),
              qw=(0.5 + torch.rand(d, generator=g, device="cuda")).to(torch.bfloat16),
              kw=(0.5 + torch.rand(d, generator=g, device="cuda")).to(torch.bfloat16),
              rope=_rope(d), q_out=torch.empty(rows, hq, d, dtype=torch.bfloat16, device="cuda"),
              slots=torch.cat([slots, torch.full((rows - total,), NO_SLOT)]).to(torch.int32).cuda(),
              positions=torch.cat([positions, torch.zeros(rows - total).long()]).to(
                  torch.int32).cuda())
    # The touched blocks, and which of them each token lies in.
    touched, which = torch.unique(slots // BLOCK, return_inverse=True)
    st.update(touched=touched.cuda(), which=which.cuda(), at=(slots % BLOCK).cuda())
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own and case["kind"] == "attention":
        from toyinfer_amd import attn
        heads = case["hq"], case["hkv"], case["d"]
        st["plan"] = attn.paged_attention_plan_buffer(case["b"], st["total"], *heads, "cuda")
        st["ws"] = attn.paged_attention_workspace(*heads, "cuda")
        # Once a step, for the attention of every layer.
        attn.paged_attention_plan(st["query_start"], st["seq_lens"], case["b"], st["total"],
                                  case["ps"], st["blocks"], case["window"], case["sinks"],
                                  *heads, st["plan"])
    return st


# -------------------------------------------------------------------- runs

def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"write": _own_write, "read": _own_read, "attention": _own_attention}[kind](st)
    return {"write": _plain_write, "read": _plain_read, "attention": _plain_attention}[kind](st)


def _own_read(st):
    from toyinfer_amd import attn
    c = st["case"]
    attn.paged_kv_read_fp8(st["k_cache"], st["v_cache"], st["tables"], st["back_start"],
                           st["seq_lens"], c["b"], st["back"], st["k_out"], st["v_out"],
                           st["pages"], c["ps"], st["k_cache"].stride(0), st["blocks"], c["hkv"],
                           c["d"])
    return st["k_out"], st["v_out"]


def _own_write(st):
    from toyinfer_amd import attn
    c = st["case"]
    attn.paged_qkv_prologue_fp8(st["q"], st["k"], st["v"], st["qw"], st["kw"], st["rope"],
                                POSITIONS, st["positions"], st["slots"], st["rows"], EPS,
                                st["q_out"], st["k_cache"], st["v_cache"], st["pages"], c["ps"],
                                st["k_cache"].stride(0), c["hq"], c["hkv"], c["d"])
    return (st["q_out"], *_own_read(st))


def _own_attention(st):
    from toyinfer_amd import attn
    c = st["case"]
    attn.paged_attention_fp8(st["q"], st["k_cache"], st["v_cache"], st["o"], st["tables"],
                             st["plan"], c["b"], st["total"], st["pages"], c["ps"],
                             st["k_cache"].stride(0), st["blocks"], c["window"], c["sinks"],
                             c["hq"], c["hkv"], c["d"], st["ws"])
    return st["o"]


def _plain_read(st):
    c, slots = st["case"], st["back_slots"]
    page, row = slots // c["ps"], slots % c["ps"]
    for cache, out in ((st["k_cache"], st["k_out"]), (st["v_cache"], st["v_out"])):
        codes = _codes(cache, c)[page, :, row].view(torch.float8_e4m3fn)
        scale = _scales(cache, c)[page, :, row // BLOCK]
        out.copy_(codes.float() * scale[..., None])
    return st["k_out"], st["v_out"]


def _plain_write(st):
    c = st["case"]
    hkv, d = c["hkv"], c["d"]
    cs = st["rope"][st["positions"].long()][:, None]  # [T][1][D/2][2]
    cos, sin = cs[..., 0], cs[..., 1]

    def rotated(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    st["q_out"].copy_(rotated(st["q"], st["qw"]))
    per_page = c["ps"] // BLOCK
    page, block = st["touched"] // per_page, st["touched"] % per_page
    rows = block[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    which, at, n = st["which"], st["at"], st["touched"].numel()
    written = torch.zeros(n, BLOCK, dtype=torch.bool, device="cuda")
    written[which, at] = True
    for cache, x in ((st["k_cache"], rotated(st["k"], st["kw"])), (st["v_cache"], st["v"].float())):
        x = x[:st["total"]]
        codes, scales = _codes(cache, c), _scales(cache, c)
        most = torch.zeros(n, BLOCK, hkv, device="cuda")
        most[which, at] = x.abs().amax(-1)
        most = most.amax(1)
        m, e = torch.frexp(most)  # m in [0.5, 1): 448 is 0.875 * 2^9
        e = (e - 9 + (m > 0.875).to(torch.int32)).clamp(LOW, HIGH)
        need = torch.ldexp(torch.ones_like(most), torch.where(most == 0, torch.full_like(e, LOW), e))
        old = scales[page, :, block]
        scale = torch.where(written[:, :1], need, torch.maximum(old, need))
        kept = codes[page[:, None], :, rows].view(torch.float8_e4m3fn).float()  # [n][16][heads][D]
        value = kept * old[:, None, :, None]
        value[which, at] = x
        value = (value / scale[:, None, :, None]).clamp(-LARGEST, LARGEST)
        codes[page[:, None], :, rows] = value.to(torch.float8_e4m3fn).view(torch.uint8)
        scales[page, :, block] = scale
    return (st["q_out"], *_plain_read(st))


def _plain_attention(st):
    c = st["case"]
    hq, hkv, d, ps = c["hq"], c["hkv"], c["d"], c["ps"]
    group, start = hq // hkv, 0

    def expanded(cache, page, L):
        codes = _codes(cache, c)[page].view(torch.float8_e4m3fn).float()
        x = codes.view(-1, hkv, ps // BLOCK, BLOCK, d) * _scales(cache, c)[page][..., None, None]
        return x.transpose(0, 1).reshape(hkv, -1, d)[:, :L]

    for b, (L, n) in enumerate(zip(st["lens"], st["fresh"])):
        if n == 0:
            continue
        page = st["tables"][b, :-(-L // ps)].long()
        k = expanded(st["k_cache"], page, L).transpose(1, 2).contiguous()
        v = expanded(st["v_cache"], page, L).contiguous()
        key = torch.arange(L, device="cuda")
        # Query rows in pieces whose scores stay around a gigabyte.
        step = max(1, (1 << 28) // (hq * L))
        for i in range(0, n, step):
            m = min(step, n - i)
            q = st["q"][start + i:start + i + m].float().view(m, hkv, group, d)
            q = q.permute(1, 2, 0, 3).reshape(hkv, group * m, d)
            s = torch.matmul(q, k).view(hkv, group, m, L) / math.sqrt(d)
            ago = (L - n + i + torch.arange(m, device="cuda"))[:, None] - key
            seen = ago >= 0
            if c["window"]:
                seen &= (ago < c["window"]) | (key < c["sinks"])
            s = s.masked_fill(~seen, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = (p / p.sum(-1, keepdim=True)).view(hkv, group * m, L)
            o = torch.matmul(p, v).view(hkv, group, m, d)
            st["o"][start + i:start + i + m] = o.permute(2, 0, 1, 3).reshape(m, hq, d).to(
                torch.bfloat16)
        start += n
    return st["o"]


# -------------------------------------------------------------------- work

def _visible(n, L, window, sinks):
    """(query, key) pairs that a request's mask leaves, and its keys that some
    query sees."""
    pairs = 0
    for p in range(L - n, L):
        w = min(window, p + 1) if window else p + 1
        pairs += w + min(sinks if window else 0, p + 1 - w)
    low = max(0, L - n - window + 1) if window else 0
    return pairs, L - low + min(sinks if window else 0, low)


def work(case):
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["ps"]
    cached, fresh = _lengths(case, 0)
    total, lens = sum(fresh), [c + n for c, n in zip(cached, fresh)]
    held = hkv * (d + 4 / BLOCK)  # bytes of a token's K or V in the cache
    if case["kind"] == "read":
        rows = sum(lens)
        return {"bytes": int(rows * (2 * held + 4 * hkv * d)) + 4 * rows // ps,
                "flops": 2 * rows * hkv * d}
    if case["kind"] == "write":
        rows = total + total // 10 if case["mix"] == "mixed" else total
        kept = sum(c % BLOCK for c, n in zip(cached, fresh) if n)
        # Q in and out, K and V in, their codes out and the blocks' earlier rows
        # in; the same rows expanded.
        return {"bytes": int(4 * rows * hq * d + 4 * rows * hkv * d + rows * (4 * d + 8)
                             + 2 * (total + kept) * held + 4 * (total + kept) * hkv * d),
                "flops": 10 * rows * d * (hq + hkv)}
    pairs = keys = 0
    for L, n in zip(lens, fresh):
        if n:
            p, k = _visible(n, L, case["window"], case["sinks"])
            pairs, keys = pairs + p, keys + k
    return {"bytes": int(4 * total * hq * d + 2 * keys * held), "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------ 64-bit values

def _held(cache, case, slots):
    """[slots][heads][dims]: what the cache holds there, by the format's bits."""
    page, row = slots // case["ps"], slots % case["ps"]
    code = _codes(cache, case)[page, :, row].long()
    exponent, fraction = code >> 3 & 15, (code & 7).double()
    size = torch.where(exponent == 0, fraction * 2.0 ** -9,
                       (1 + fraction / 8) * torch.exp2(exponent.double() - 7))
    scale = _scales(cache, case)[page, :, row // BLOCK].double()
    return torch.where(code >> 7 == 1, -size, size) * scale[..., None]


def _nearest(x):
    """x to four significant bits, halves to even, in steps of 2^-9 at least."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return torch.round(x / step).mul(step).clamp(-LARGEST, LARGEST)


def _exact_write(case, st):
    hkv, d, half = case["hkv"], case["d"], case["d"] // 2
    angle = st["rope"].double()[st["positions"].long()]

    def turned(x, w):
        x = x.double()
        x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        y = torch.empty_like(x)
        c, s = angle[:, None, :, 0], angle[:, None, :, 1]
        y[..., :half] = x[..., :half] * c - x[..., half:] * s
        y[..., half:] = x[..., half:] * c + x[..., :half] * s
        return y

    n, index = st["touched"].numel(), st["which"] * BLOCK + st["at"]
    slots = (st["touched"][:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).reshape(-1)
    rows = torch.full((st["pages"] * case["ps"],), -1, dtype=torch.long, device="cuda")
    rows[slots] = torch.arange(slots.numel(), device="cuda")
    live = st["slots"] >= 0
    fresh = torch.zeros(n * BLOCK, dtype=torch.bool, device="cuda")
    fresh[index] = True
    outs = [turned(st["q"], st["qw"])]
    for cache, x in ((st["k_cache"], turned(st["k"], st["kw"])), (st["v_cache"], st["v"].double())):
        new = torch.zeros(n * BLOCK, hkv, d, dtype=torch.float64, device="cuda")
        new[index] = x[live]
        most = new.abs().view(n, BLOCK, hkv, d).amax((1, 3))
        scale = torch.exp2(torch.ceil(torch.log2(most / LARGEST)).clamp(LOW, HIGH))
        scale = torch.where(most > LARGEST * scale, 2 * scale, scale)  # (the logarithm's rounding)
        first = slots[::BLOCK]
        before = _scales(cache, case)[first // case["ps"], :, first % case["ps"] // BLOCK].double()
        scale = torch.where(fresh.view(n, BLOCK)[:, :1], scale, torch.maximum(scale, before))
        scale = scale.repeat_interleave(BLOCK, 0)[..., None]
        value = torch.where(fresh[:, None, None], new, _held(cache, case, slots))
        outs.append((_nearest(value / scale) * scale)[rows[st["back_slots"]]])
    return tuple(outs)


def exact(case, seed):
    st = _inputs(case, seed)
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["ps"]
    if case["kind"] == "read":
        return tuple(_held(st[x], case, st["back_slots"]) for x in ("k_cache", "v_cache"))
    if case["kind"] == "write":
        return _exact_write(case, st)
    out = torch.zeros(st["total"], hq, d, dtype=torch.float64, device="cuda")
    first = 0
    for b in range(case["b"]):
        L, n = st["lens"][b], st["fresh"][b]
        where = torch.arange(L, device="cuda")
        slot = st["tables"][b].long()[where // ps] * ps + where % ps
        keys, values = _held(st["k_cache"], case, slot), _held(st["v_cache"], case, slot)
        for h in range(hkv if n else 0):
            k, v = keys[:, h].t().contiguous(), values[:, h].contiguous()
            for head in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                for i in range(0, n, 4096):
                    rows = slice(first + i, first + min(n, i + 4096))
                    p = L - n + torch.arange(i, min(n, i + 4096), device="cuda")[:, None]
                    hidden = where > p
                    if case["window"]:
                        hidden |= (where <= p - case["window"]) & (where >= case["sinks"])
                    s = (st["q"][rows, head].double() @ k) * d ** -0.5
                    out[rows, head] = s.masked_fill(hidden, -math.inf).softmax(-1) @ v
        first += n
    return out
