"""Performance cases of the paged-cache operators: serving many requests at once.

One step of a server takes a batch of requests, each with tokens already in the
cache and new ones (a decoded token, a chunk of a prompt, a whole prompt):
`tables` gives the new tokens pages and slots, `prologue` normalises and rotates
one layer's Q and K and writes K and V to the slots, `attention` runs the new
tokens over the pages.  With `own` false `run` computes the same in elementary
torch operations; `exact` gives the results in 64 bits.
"""
import math

import torch

own = False

EPS, THETA = 1e-6, 1e6
NO_SLOT = -1  # 0xFFFFFFFF as the int32 that torch holds


def listed():
    return [
        # A decode step of eight requests: launch-bound bookkeeping.
        {"name": "tables_decode_b8", "kind": "tables", "mix": "decode", "b": 8, "new": 1,
         "ctx": 4096, "ps": 16, "hq": 16, "hkv": 8, "d": 128},
        # A step of a loaded server: decoding requests beside prompts in chunks,
        # rows for tokens that this step does not fill.
        {"name": "tables_mixed_b200", "kind": "tables", "mix": "mixed", "b": 200, "new": 512,
         "ctx": 8192, "ps": 16, "hq": 32, "hkv": 8, "d": 128},
        # One token of eight requests, Qwen3-8B heads.
        {"name": "prologue_t8", "kind": "prologue", "t": 8, "ps": 16, "hq": 32, "hkv": 8, "d": 128},
        # A chat prompt, Qwen3-0.6B heads.
        {"name": "prologue_t1371", "kind": "prologue", "t": 1371, "ps": 16, "hq": 16, "hkv": 8,
         "d": 128},
        # Prompts of 8192 tokens in all.
        {"name": "prologue_t8192", "kind": "prologue", "t": 8192, "ps": 64, "hq": 32, "hkv": 8,
         "d": 128},
        # The next token of one chat: latency.
        {"name": "decode_b1_l1371", "kind": "attention", "mix": "decode", "b": 1, "new": 1,
         "ctx": 1371, "ps": 16, "window": 0, "sinks": 0, "hq": 16, "hkv": 8, "d": 128},
        # The next token of 32 requests of different lengths.
        {"name": "decode_b32_l8192", "kind": "attention", "mix": "decode", "b": 32, "new": 1,
         "ctx": 8192, "ps": 16, "window": 0, "sinks": 0, "hq": 32, "hkv": 8, "d": 128},
        # The same deep in long conversations under a window with four sinks.
        {"name": "decode_b16_window", "kind": "attention", "mix": "decode", "b": 16, "new": 1,
         "ctx": 32768, "ps": 64, "window": 4096, "sinks": 4, "hq": 32, "hkv": 8, "d": 128},
        # The next piece of one long prompt.
        {"name": "chunk_t512_l8192", "kind": "attention", "mix": "chunk", "b": 1, "new": 512,
         "ctx": 7680, "ps": 16, "window": 0, "sinks": 0, "hq": 32, "hkv": 8, "d": 128},
        # Decoding requests and a few prompt pieces in one batch, head_dim 64.
        {"name": "mixed_b24_d64", "kind": "attention", "mix": "mixed", "b": 24, "new": 300,
         "ctx": 3000, "ps": 32, "window": 0, "sinks": 0, "hq": 32, "hkv": 8, "d": 64},
        # A piece of a prompt under a window, an odd group of heads.
        {"name": "chunk_window_g3", "kind": "attention", "mix": "chunk", "b": 3, "new": 777,
         "ctx": 5000, "ps": 16, "window": 1024, "sinks": 16, "hq": 6, "hkv": 2, "d": 128},
        # A whole long prompt into empty pages.
        {"name": "prompt_t8192", "kind": "attention", "mix": "chunk", "b": 1, "new": 8192,
         "ctx": 0, "ps": 16, "window": 0, "sinks": 0, "hq": 32, "hkv": 8, "d": 128},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "prologue", "attention", "attention", "attention"])
    hq, hkv = rng.choice([(16, 8), (32, 8), (8, 8), (12, 2), (6, 2), (5, 1), (28, 4)])
    c = {"kind": kind, "ps": rng.choice([8, 16, 16, 32, 64, 128, 256]), "hq": hq, "hkv": hkv,
         "d": rng.choice([128, 128, 64])}
    if kind == "prologue":
        c["t"] = _log_int(rng, 1, 8192)
        return c
    c["mix"] = rng.choice(["decode", "chunk", "mixed"])
    if kind == "tables":
        c["b"] = _log_int(rng, 1, 256)
        c["new"] = 1 if c["mix"] == "decode" else _log_int(rng, 2, 16384 // c["b"] + 2)
        c["ctx"] = _log_int(rng, 1, 8192)
        return c
    # At most the longest listed prompt's products (new tokens times context)
    # and its cache times eight.
    c["b"] = _log_int(rng, 1, 48 if c["mix"] == "decode" else 24)
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
    chunk, one in sixteen idle, the others one token.  The seed orders them and
    says how much of `ctx` each has cached."""
    b, new, ctx = case["b"], case["new"], case["ctx"]
    r = torch.Generator().manual_seed(seed)
    u = torch.rand(b, generator=r).tolist()
    cached = [ctx - int(0.75 * ctx * x) if i else ctx for i, x in enumerate(u)]
    fresh = []
    for i in range(b):
        if case["mix"] == "decode":
            fresh.append(new)
        elif case["mix"] == "chunk" or i % 8 == 0:
            fresh.append(new - new // 2 * i // b)
        else:
            fresh.append(0 if i % 16 == 9 else 1)
    return cached, [fresh[i] for i in torch.randperm(b, generator=r).tolist()]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rope(positions, d):
    inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float()


def _starts(n):
    s = [0]
    for x in n:
        s.append(s[-1] + x)
    return s


def _inputs(case, seed):
    """What a case reads and the buffers it writes, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = torch.Generator().manual_seed(seed)
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["ps"]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)

    st = {"case": case}
    if case["kind"] == "prologue":
        t = case["t"]
        pages = 2 * (-(-t // ps)) + 1
        i = torch.arange(t)
        slots = torch.randperm(pages, generator=r)[i // ps] * ps + i % ps
        # A few tokens are of as many requests, more are one prompt's.
        positions = (torch.randint(0, 40960, (t,), generator=r) if t <= 64
                     else torch.randint(0, 40960 - t, (1,), generator=r) + i)
        st.update(q=normal(t, hq, d, std=2.0), k=normal(t, hkv, d, std=2.0), v=normal(t, hkv, d),
                  qw=(0.5 + torch.rand(d, generator=g, device="cuda")).to(torch.bfloat16),
                  kw=(0.5 + torch.rand(d, generator=g, device="cuda")).to(torch.bfloat16),
                  rope=_rope(40960, d), slots=slots.to(torch.int32).cuda(),
                  positions=positions.to(torch.int32).cuda(),
                  k_cache=normal(pages, ps, hkv, d), v_cache=normal(pages, ps, hkv, d),
                  q_out=torch.empty(t, hq, d, dtype=torch.bfloat16, device="cuda"))
        return st
    cached, fresh = _lengths(case, seed)
    total = sum(fresh)
    if case["kind"] == "tables":
        # Pages of the cached tokens are in the tables, the rest on the stack
        # of free ones; a tenth more token rows than this step fills.
        blocks = -(-(case["ctx"] + case["new"]) // ps) + 1
        used = [-(-c // ps) for c in cached]
        need = sum(-(-(c + n) // ps) for c, n in zip(cached, fresh)) - sum(used)
        order = torch.randperm(sum(used) + need + 16, generator=r).to(torch.int32)
        tables = torch.full((case["b"], blocks), NO_SLOT, dtype=torch.int32)
        for i, s in enumerate(_starts(used)[:-1]):
            tables[i, :used[i]] = order[s:s + used[i]]
        rows = total + total // 10
        free = order[sum(used):]
        st.update(context_lens=_ints(cached), new_lens=_ints(fresh), tables=tables.cuda(),
                  free=free.cuda(), num_free=_ints([free.numel()]), blocks=blocks, rows=rows,
                  query_start=_ints([0] * (case["b"] + 1)), seq_lens=_ints([0] * case["b"]),
                  positions=_ints([0] * rows), slots=_ints([0] * rows), status=_ints([0, 0]))
        return st
    lens = [c + n for c, n in zip(cached, fresh)]
    used = [-(-x // ps) for x in lens]
    blocks = max(used) + 1
    pages = sum(used) + 7
    order = torch.randperm(pages, generator=r).to(torch.int32)
    tables = torch.full((case["b"], blocks), NO_SLOT, dtype=torch.int32)
    for i, s in enumerate(_starts(used)[:-1]):
        tables[i, :used[i]] = order[s:s + used[i]]
    st.update(lens=lens, fresh=fresh, total=total, blocks=blocks, pages=pages,
              q=normal(total, hq, d, std=1.5), k_cache=normal(pages, ps, hkv, d),
              v_cache=normal(pages, ps, hkv, d), tables=tables.cuda(),
              seq_lens=_ints(lens), query_start=_ints(_starts(fresh)),
              o=torch.empty(total, hq, d, dtype=torch.bfloat16, device="cuda"))
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own and case["kind"] != "prologue":
        from toyinfer_amd import attn
        heads = case["hq"], case["hkv"], case["d"]
        rows = st["rows"] if case["kind"] == "tables" else st["total"]
        st["plan"] = attn.paged_attention_plan_buffer(case["b"], rows, *heads, "cuda")
        if case["kind"] == "attention":
            st["ws"] = attn.paged_attention_workspace(*heads, "cuda")
            # Once a step, for the attention of every layer.
            attn.paged_attention_plan(st["query_start"], st["seq_lens"], case["b"], rows,
                                      case["ps"], st["blocks"], case["window"], case["sinks"],
                                      *heads, st["plan"])
    return st


# -------------------------------------------------------------------- runs

def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"tables": _own_tables, "prologue": _own_prologue,
                "attention": _own_attention}[kind](st)
    return {"tables": _plain_tables, "prologue": _plain_prologue,
            "attention": _plain_attention}[kind](st)


def _tables_out(st):
    return {k: st[k] for k in ("query_start", "seq_lens", "positions", "slots", "tables", "status")}


def _own_tables(st):
    """All that a step prepares once for its layers: tables, slots, positions
    and the attention's plan."""
    from toyinfer_amd import attn
    c = st["case"]
    attn.paged_tables_u32(st["context_lens"], st["new_lens"], c["b"], st["free"],
                          st["free"].numel(), st["num_free"], c["ps"], st["tables"], st["blocks"],
                          st["rows"], st["query_start"], st["seq_lens"], st["positions"],
                          st["slots"], st["status"])
    attn.paged_attention_plan(st["query_start"], st["seq_lens"], c["b"], st["rows"], c["ps"],
                              st["blocks"], 0, 0, c["hq"], c["hkv"], c["d"], st["plan"])
    return _tables_out(st)


def _plain_tables(st):
    c, ps, rows = st["case"], st["case"]["ps"], st["rows"]
    b = c["b"]
    ctx, new = st["context_lens"].long(), st["new_lens"].long()
    old, end = (ctx + ps - 1) // ps, (ctx + new + ps - 1) // ps
    need = torch.where(end <= st["blocks"], end - old, torch.zeros_like(end))
    upto = need.cumsum(0)
    ok = ((need == 0) | (upto <= st["num_free"].long())) & (end <= st["blocks"])
    need = torch.where(ok, need, torch.zeros_like(need))
    first = upto - (end - old)
    j = torch.arange(st["blocks"], device="cuda")[None, :]
    fresh = ok[:, None] & (j >= old[:, None]) & (j < end[:, None])
    at = st["num_free"].long() - 1 - (first[:, None] + j - old[:, None])
    page = st["free"][at.clamp(0, st["free"].numel() - 1)]
    st["tables"].copy_(torch.where(fresh, page, st["tables"]))
    ends = new.cumsum(0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    t = torch.arange(rows, device="cuda")
    req = torch.searchsorted(ends, t, right=True)
    live = req < b
    req = req.clamp(max=b - 1)
    pos = ctx[req] + t - starts[req]
    live_slot = live & ok[req]
    entry = st["tables"][req, (pos // ps).clamp(0, st["blocks"] - 1)].long()
    st["query_start"].copy_(starts)
    st["seq_lens"].copy_(torch.where(ok, ctx + new, ctx))
    st["positions"].copy_(torch.where(live, pos, torch.zeros_like(pos)))
    st["slots"].copy_(torch.where(live_slot, entry * ps + pos % ps, torch.full_like(pos, NO_SLOT)))
    st["status"].copy_(torch.stack([st["num_free"][0].long() - need.sum(), (~ok).sum()]))
    return _tables_out(st)


def _own_prologue(st):
    from toyinfer_amd import attn
    c = st["case"]
    pages = st["k_cache"].shape[0]
    attn.paged_qkv_prologue_bf16(st["q"], st["k"], st["v"], st["qw"], st["kw"], st["rope"], 40960,
                                 st["positions"], st["slots"], c["t"], EPS, st["q_out"],
                                 st["k_cache"], st["v_cache"], pages, c["ps"],
                                 c["ps"] * c["hkv"] * c["d"], c["hq"], c["hkv"], c["d"])
    return st["q_out"], st["k_cache"], st["v_cache"]


def _plain_prologue(st):
    c = st["case"]
    hkv, d = c["hkv"], c["d"]
    cs = st["rope"][st["positions"].long()][:, None]  # [T][1][D/2][2]
    cos, sin = cs[..., 0], cs[..., 1]

    def rotated(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(torch.bfloat16)

    slots = st["slots"].long()
    st["q_out"].copy_(rotated(st["q"], st["qw"]))
    st["k_cache"].view(-1, hkv, d)[slots] = rotated(st["k"], st["kw"])
    st["v_cache"].view(-1, hkv, d)[slots] = st["v"]
    return st["q_out"], st["k_cache"], st["v_cache"]


def _own_attention(st):
    from toyinfer_amd import attn
    c = st["case"]
    attn.paged_attention_bf16(st["q"], st["k_cache"], st["v_cache"], st["o"], st["tables"],
                              st["plan"], c["b"], st["total"], st["pages"], c["ps"],
                              c["ps"] * c["hkv"] * c["d"], st["blocks"], c["window"], c["sinks"],
                              c["hq"], c["hkv"], c["d"], st["ws"])
    return st["o"]


def _plain_attention(st):
    c = st["case"]
    hq, hkv, d, ps = c["hq"], c["hkv"], c["d"], c["ps"]
    group, start = hq // hkv, 0
    for b, (L, n) in enumerate(zip(st["lens"], st["fresh"])):
        if n == 0:
            continue
        page = st["tables"][b, :-(-L // ps)].long()
        k = st["k_cache"][page].view(-1, hkv, d)[:L].float().permute(1, 2, 0).contiguous()
        v = st["v_cache"][page].view(-1, hkv, d)[:L].float().transpose(0, 1).contiguous()
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
    if case["kind"] == "prologue":
        t = case["t"]
        return {"bytes": 2 * t * d * (2 * hq + 4 * hkv) + t * (4 * d + 8) + 4 * d,
                "flops": 10 * t * d * (hq + hkv)}
    cached, fresh = _lengths(case, 0)
    if case["kind"] == "tables":
        total = sum(fresh)
        rows = total + total // 10
        pages = sum(-(-(c + n) // ps) - -(-c // ps) for c, n in zip(cached, fresh))
        # Lengths in and out, pages off the stack into the tables, the entry of
        # each page that a token lies in, position and slot per token row.
        return {"bytes": 16 * case["b"] + 8 * pages + 4 * max(total // ps, case["b"]) + 8 * rows,
                "flops": 4 * rows}
    pairs = keys = 0
    for c, n in zip(cached, fresh):
        if n:
            p, k = _visible(n, c + n, case["window"], case["sinks"])
            pairs, keys = pairs + p, keys + k
    return {"bytes": 4 * sum(fresh) * hq * d + 4 * keys * hkv * d, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------ 64-bit values

def exact(case, seed):
    if case["kind"] == "tables":
        return None  # whole numbers
    st = _inputs(case, seed)
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["ps"]
    if case["kind"] == "prologue":
        half = d // 2
        angle = st["rope"].double()[st["positions"].long()]

        def turned(x, w):
            x = x.double()
            x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
            y = torch.empty_like(x)
            c, s = angle[:, None, :, 0], angle[:, None, :, 1]
            y[..., :half] = x[..., :half] * c - x[..., half:] * s
            y[..., half:] = x[..., half:] * c + x[..., :half] * s
            return y

        k_cache = st["k_cache"].double().reshape(-1, hkv, d)
        v_cache = st["v_cache"].double().reshape(-1, hkv, d)
        k_cache.index_copy_(0, st["slots"].long(), turned(st["k"], st["kw"]))
        v_cache.index_copy_(0, st["slots"].long(), st["v"].double())
        return (turned(st["q"], st["qw"]), k_cache.view(st["k_cache"].shape),
                v_cache.view(st["v_cache"].shape))
    out = torch.zeros(st["total"], hq, d, dtype=torch.float64, device="cuda")
    first = 0
    for b in range(case["b"]):
        L, n = st["lens"][b], st["fresh"][b]
        where = torch.arange(L, device="cuda")
        slot = st["tables"][b].long()[where // ps] * ps + where % ps
        for h in range(hkv):
            k = st["k_cache"].view(-1, hkv, d)[slot, h].double().t().contiguous()
            v = st["v_cache"].view(-1, hkv, d)[slot, h].double()
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
