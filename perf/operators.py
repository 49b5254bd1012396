"""Attention over keys that several rows share, and the append that feeds it, as measurable cases.

Three operators of a server's decoder layers, through vm_c_amd.capi (the C
ABI's entry points), inputs resident in GPU memory:

  prefix  one new token per sequence over a paged cache whose sequences come in
          groups with a common prefix (a system prompt, a document, the samples
          of one prompt): the prefix's keys are read once for the group.
          f16 / bf16 / q8_0 / q4_0 pages; head_dim 64, 128 and 256.
  cross   rows of a decoder over an encoder's states of another length, no
          causal mask: whole targets, single tokens, or the hypotheses of one
          input, which share its states.
  rope    the position rotation of Q and K, read from the fused QKV projection,
          and the append of K and V to the paged cache in the same pass.

Values are N(0, 1) before quantization; block tables are permutations of a
shared pool; prefixes are whole pages, as a block manager shares them.
"""
import math

import numpy as np
import torch

own = False

BS = 16  # tokens per page
_DT = {"f16": torch.float16, "bf16": torch.bfloat16}
_PAGES = {"fp16": "f16", "bf16": "bf16"}  # page formats that hold 16-bit values
MAX_POS = 32768  # rows of the rotation table


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # A few chat turns behind one short system prompt: the smallest call, bound by launches and latency.
        _prefix("prefix_f16_b4", fmt="fp16", groups="4x512", lo=1, hi=100, len_seed=1),
        # Sixteen samples of one prompt over GGUF pages, each a few hundred tokens along.
        _prefix("prefix_q8_0_b16", fmt="q8_0", dtype="bf16", groups="16x4096", lo=1, hi=1000, len_seed=2),
        # Many users of one long document: the largest, 64 rows over 32768 shared tokens.
        _prefix("prefix_bf16_b64_32k", fmt="bf16", dtype="bf16", groups="64x32768", lo=32, hi=2048, len_seed=3),
        # Four tenants with a system prompt each, head_dim 256, 4-bit pages by head.
        _prefix("prefix_q4_0_d256_4groups", fmt="q4_0", groups="13x1008 3x8192 9x2000 7x16384",
                hq=16, hkv=2, d=256, layout="hnd", lo=17, hi=700, len_seed=4),
        # A small model's batch: two groups, and rows that share nothing.
        _prefix("prefix_bf16_d64_b48", fmt="bf16", dtype="bf16", groups="21x6000 1x0 1x0 25x3008", d=64, lo=64, hi=4096,
                len_seed=5),
        # Single target tokens of eight inputs of 1500 states each (an audio window), a head of its own per query head.
        _cross("cross_f16_b8_decode", dtype="f16", batch=8, t_lo=1, t_hi=1, n_lo=1500, n_hi=1500, hq=16, hkv=16, d=64),
        # Five hypotheses each of 32 documents, ragged encoder lengths: one token of every hypothesis.
        _cross("cross_bf16_b32_beams", dtype="bf16", batch=32, t_lo=5, t_hi=5, n_lo=200, n_hi=4096, hq=32, hkv=8, d=128,
               len_seed=6),
        # Whole targets against whole inputs: eight of 1024 tokens over 2048 states, bound by the products.
        _cross("cross_bf16_8x1024", dtype="bf16", batch=8, t_lo=1024, t_hi=1024, n_lo=2048, n_hi=2048, hq=32, hkv=8,
               d=128),
        # Short ragged targets over short ragged inputs, one head_dim 64 head each.
        _cross("cross_f16_ragged", dtype="f16", batch=24, t_lo=9, t_hi=333, n_lo=31, n_hi=1500, hq=12, hkv=12, d=64,
               len_seed=7),
        # A decode step's 32 tokens: rotation and append, bound by one launch.
        _rope("rope_bf16_b32", dtype="bf16", tokens=32),
        # A prefill step of a small model, interleaved pairs, pages by head, an odd number of tokens.
        _rope("rope_f16_d64_5k", dtype="f16", tokens=5003, hq=14, hkv=2, d=64, rot=64, neox=False, layout="hnd"),
        # A large prefill step of the head_dim 256 deployment, which rotates a quarter of a head.
        _rope("rope_bf16_d256_16k", dtype="bf16", tokens=16384, hq=16, hkv=2, d=256, rot=64),
    ]


def _prefix(name, *, fmt, groups, lo, hi, hq=32, hkv=8, d=128, dtype="f16", layout="nhd", len_seed=0):
    """groups: rows x shared tokens of each; lo .. hi: tokens of a row past its prefix."""
    return _named(name, kind="prefix", fmt=fmt, groups=groups, hq=hq, hkv=hkv, d=d, dtype=dtype, layout=layout, lo=lo,
                  hi=hi, len_seed=len_seed)


def _cross(name, *, dtype, batch, t_lo, t_hi, n_lo, n_hi, hq, hkv, d, len_seed=0):
    return _named(name, kind="cross", dtype=dtype, batch=batch, t_lo=t_lo, t_hi=t_hi, n_lo=n_lo, n_hi=n_hi, hq=hq,
                  hkv=hkv, d=d, len_seed=len_seed)


def _rope(name, *, dtype, tokens, hq=32, hkv=8, d=128, rot=128, neox=True, layout="nhd"):
    return _named(name, kind="rope", dtype=dtype, tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, neox=neox,
                  layout=layout)


def _named(name, **case):
    return dict(case, name=name) if name else case


def draw(rng):
    """Another call of the same families; lengths and batches are spread over
    their logarithm, and a call that would pass the largest listed one is cut."""
    kind = rng.choice(["prefix", "prefix", "cross", "cross", "rope"])
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))  # noqa: E731
    len_seed = rng.randrange(1 << 20)
    if kind == "prefix":
        d = rng.choice([64, 128, 128, 256])
        hq, hkv = rng.choice({64: [(32, 8), (14, 2)], 128: [(32, 8), (64, 8), (28, 4), (16, 2)],
                              256: [(16, 2), (8, 4)]}[d])
        fmt = rng.choice(["fp16", "bf16", "q8_0", "q4_0"])
        groups, rows, tokens = [], 0, 0
        for _ in range(rng.choice([1, 1, 2, 3, 5])):
            n = min(log(1, 64), 64 - rows)
            shared = BS * log(1, 2048)
            if n < 1 or (tokens + n * shared) * hkv * d > 64 * 32768 * 1024 or (hq == 64 and n * shared > 32 * 32768):
                continue
            groups.append(f"{n}x{shared}")
            rows, tokens = rows + n, tokens + n * shared
        groups = " ".join(groups) or f"{log(2, 16)}x1024"
        hi = log(1, 2048)
        return _prefix("", fmt=fmt, groups=groups, hq=hq, hkv=hkv, d=d, lo=max(1, hi // 16), hi=hi,
                       dtype=_PAGES.get(fmt) or rng.choice(["f16", "bf16"]), layout=rng.choice(["nhd", "nhd", "hnd"]),
                       len_seed=len_seed)
    dtype = rng.choice(["f16", "bf16"])
    if kind == "cross":
        d = rng.choice([64, 128, 128, 256])
        hq, hkv = rng.choice({64: [(16, 16), (12, 12), (32, 8)], 128: [(32, 8), (16, 16), (28, 4)],
                              256: [(16, 2), (8, 8)]}[d])
        t_hi = rng.choice([1, 1, log(2, 16), log(2, 1024)])
        n_hi = log(16, 4096)
        room = 8 * 1024 * 2048 * 32 * 128 // (t_hi * n_hi * hq * d)
        batch = max(1, min(log(1, 64), room, 24 * 4096 * 1024 // (n_hi * hkv * d), 16384 // t_hi))
        return _cross("", dtype=dtype, batch=batch, t_lo=max(1, t_hi // 8), t_hi=t_hi, n_lo=max(1, n_hi // 8),
                      n_hi=n_hi, hq=hq, hkv=hkv, d=d, len_seed=len_seed)
    d = rng.choice([64, 128, 256])
    hq, hkv = rng.choice({64: [(14, 2), (12, 12)], 128: [(32, 8), (28, 4)], 256: [(16, 2), (8, 4)]}[d])
    return _rope("", dtype=dtype, tokens=log(1, 15000 * 5120 // ((hq + 2 * hkv) * d)), hq=hq, hkv=hkv, d=d,
                 rot=rng.choice([d, d, d // 2, d // 4]), neox=rng.random() < 0.7, layout=rng.choice(["nhd", "hnd"]))


def _spread(seed, lo, hi, n):
    """n lengths from lo to hi, evenly over the logarithm; the first is the longest."""
    rng = np.random.default_rng(seed)
    x = np.exp(rng.uniform(math.log(lo), math.log(hi), n)).astype(np.int64)
    x[0] = hi
    return np.clip(x, lo, hi)


def _groups(c):
    """Rows and shared tokens of each group."""
    return np.array([g.split("x") for g in c["groups"].split()], np.int64).T


def _prefix_lens(c):
    """(rows of each group, shared tokens of each row, tokens of each row)."""
    rows, shared = _groups(c)
    shared = np.repeat(shared, rows)
    return rows, shared, shared + _spread(c["len_seed"], c["lo"], c["hi"], int(rows.sum()))


def _cross_lens(c):
    return (_spread(c["len_seed"] + 1, c["t_lo"], c["t_hi"], c["batch"]),
            _spread(c["len_seed"] + 2, c["n_lo"], c["n_hi"], c["batch"]))


# ------------------------------------------------------------------ page formats, in plain torch

def _entry_bytes(fmt, d):
    return {"fp16": 2 * d, "bf16": 2 * d, "q8_0": 34 * (d // 32), "q4_0": 18 * (d // 32)}[fmt]


def _encode_page(x, fmt):
    """[.., d] values -> page entries, as bytes."""
    if fmt in _PAGES:
        return x.to(_DT[_PAGES[fmt]]).view(torch.uint8)
    x = x.view(*x.shape[:-1], -1, 32)
    if fmt == "q8_0":
        s = x.abs().amax(-1, keepdim=True) / 127
        q = torch.round(x / s.clamp_min(1e-30)).to(torch.int8).view(torch.uint8)
    else:
        big = x.gather(-1, x.abs().argmax(-1, keepdim=True))
        s = big / -8
        q = (x / torch.where(s == 0, torch.ones_like(s), s) + 8.5).to(torch.int32).clamp_(0, 15)
        q = (q[..., :16] | (q[..., 16:] << 4)).to(torch.uint8)
    return torch.cat([s.to(torch.float16).view(torch.uint8), q], -1).flatten(-2)


def _decode_page(b, fmt, to):
    """Page entries -> the values they stand for."""
    if fmt in _PAGES:
        return b.contiguous().view(_DT[_PAGES[fmt]]).to(to)
    b = b.view(*b.shape[:-1], -1, 34 if fmt == "q8_0" else 18)
    s = b[..., :2].contiguous().view(torch.float16).to(to)
    if fmt == "q8_0":
        q = b[..., 2:].contiguous().view(torch.int8).to(to)
    else:
        q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).to(to) - 8
    return (q * s).flatten(-2)


def _tokens_first(pool, c):
    """A pool as [page][token][kv head][entry]."""
    e = _entry_bytes(c["fmt"], c["d"])
    if c["layout"] == "hnd":
        return pool.view(-1, c["hkv"], BS, e).transpose(1, 2)
    return pool.view(-1, BS, c["hkv"], e)


# ------------------------------------------------------------------ inputs

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case, "scale": 1.0 / math.sqrt(case["d"])}
    {"prefix": _prepare_prefix, "cross": _prepare_cross, "rope": _prepare_rope}[case["kind"]](s, case, g)
    return s


def _prepare_prefix(s, c, g):
    rows, shared, lens = _prefix_lens(c)
    hq, hkv, d, dt = c["hq"], c["hkv"], c["d"], _DT[c["dtype"]]
    first = np.repeat(np.concatenate([[0], np.cumsum(rows)[:-1]]), rows)  # each row's group's first row
    n_pages, n_shared = (lens + BS - 1) // BS, shared // BS
    private = n_pages - np.where(first == np.arange(len(lens)), 0, n_shared)  # pages of a row's own
    at = np.concatenate([[0], np.cumsum(private)])
    order = torch.randperm(int(at[-1]), generator=g, device="cuda").cpu().numpy()
    bt = np.full((len(lens), int(n_pages.max())), -1, np.int64)
    for b in range(len(lens)):
        mine = order[at[b]:at[b + 1]]
        bt[b, n_pages[b] - len(mine):n_pages[b]] = mine
        bt[b, :n_pages[b] - len(mine)] = bt[first[b], :n_pages[b] - len(mine)]
    s["bt"], s["lens"] = _dev(bt), _dev(lens)
    s["group_starts"] = _dev(np.concatenate([[0], np.cumsum(rows)]))
    s["shared_lens"] = _dev(_groups(c)[1])
    n, e = int(at[-1]) * BS * hkv, _entry_bytes(c["fmt"], d)
    for name in ("k_pool", "v_pool"):
        pool = torch.empty((n, e), dtype=torch.uint8, device="cuda")
        for i in range(0, n, 1 << 19):
            m = min(1 << 19, n - i)
            pool[i:i + m] = _encode_page(_randn(g, m, d), c["fmt"])
        s[name] = pool.view(-1)
    s["q"] = _randn(g, len(lens), hq, d, dtype=dt)
    s["out"] = torch.empty_like(s["q"])
    if own:
        from vm_c_amd import capi
        s["ws"] = torch.empty(capi.shared_prefix_workspace_size(len(lens), hq, hkv, d, len(rows)), dtype=torch.uint8,
                              device="cuda")


def _prepare_cross(s, c, g):
    t, n = _cross_lens(c)
    hq, hkv, d, dt = c["hq"], c["hkv"], c["d"], _DT[c["dtype"]]
    s["q_starts"] = _dev(np.concatenate([[0], np.cumsum(t)]))
    s["k_starts"] = _dev(np.concatenate([[0], np.cumsum(n)[:-1]]))
    s["k_lens"] = _dev(n)
    s["q"] = _randn(g, int(t.sum()), hq, d, dtype=dt)
    kv = _randn(g, int(n.sum()), 2, hkv, d, dtype=dt)  # the states' fused K and V projection
    s["k"], s["v"] = kv[:, 0], kv[:, 1]
    s["out"] = torch.empty_like(s["q"])
    if own:
        from vm_c_amd import capi
        s["ws"] = torch.empty(capi.cross_attention_workspace_size(len(s["q"]), len(t), hq, hkv, d), dtype=torch.uint8,
                              device="cuda")


def _prepare_rope(s, c, g):
    t, hq, hkv, d, dt = c["tokens"], c["hq"], c["hkv"], c["d"], _DT[c["dtype"]]
    qkv = _randn(g, t, hq + 2 * hkv, d, dtype=dt)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    half = c["rot"] // 2
    ang = torch.arange(MAX_POS, device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).float()
    s["pos"] = torch.randint(0, MAX_POS, (t,), generator=g, device="cuda")
    pages = (t + BS - 1) // BS
    page = torch.randperm(pages, generator=g, device="cuda")
    at = torch.arange(t, device="cuda")
    s["slots"] = page[at // BS] * BS + at % BS
    shape = (pages, BS, hkv, d) if c["layout"] == "nhd" else (pages, hkv, BS, d)
    s["k_pool"], s["v_pool"] = (torch.zeros(shape, dtype=dt, device="cuda") for _ in range(2))
    s["q_out"] = torch.empty((t, hq, d), dtype=dt, device="cuda")


# ------------------------------------------------------------------ one pass

def run(state):
    s = state
    if own:
        return {"prefix": _own_prefix, "cross": _own_cross, "rope": _own_rope}[s["case"]["kind"]](s)
    return {"prefix": _plain_prefix, "cross": _plain_cross, "rope": _plain_rope}[s["case"]["kind"]](s)


def _own_prefix(s):
    from vm_c_amd import capi
    c = s["case"]
    return capi.paged_attention_shared_prefix(
        s["out"], s["q"], s["k_pool"], s["v_pool"], s["bt"], s["lens"], s["group_starts"], s["shared_lens"], c["hkv"],
        s["scale"], block_size=BS, kv_format=capi.KV_FORMATS[c["fmt"]],
        layout=capi.LAYOUT_HND if c["layout"] == "hnd" else capi.LAYOUT_NHD, workspace=s["ws"])


def _own_cross(s):
    from vm_c_amd import capi
    return capi.cross_attention(s["out"], s["q"], s["k"], s["v"], s["q_starts"], s["k_starts"], s["k_lens"], s["scale"],
                                workspace=s["ws"])


def _own_rope(s):
    from vm_c_amd import capi
    c = s["case"]
    capi.rope_and_cache(s["q"], s["k"], s["v"], s["cos_sin"], s["pos"], s["k_pool"], s["v_pool"], s["slots"], BS,
                        query_out=s["q_out"], is_neox=c["neox"],
                        kv_format=capi.KV_FORMATS["fp16" if c["dtype"] == "f16" else "bf16"],
                        layout=capi.LAYOUT_HND if c["layout"] == "hnd" else capi.LAYOUT_NHD)
    return s["q_out"], s["k_pool"], s["v_pool"]


def _attend_plain(q, k, v, there, scale):
    """q [b][h][r][d] over k, v [b][h][n][d] where `there` [b][1][1][n], in 32 bits."""
    x = torch.matmul(q, k.transpose(-1, -2)) * scale
    x = torch.where(there, x, torch.full_like(x, -math.inf))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return torch.matmul(x, v) / x.sum(-1, keepdim=True)


def _plain_prefix(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    b, m = s["bt"].shape
    table = s["bt"].clamp_min(0).long()
    k, v = (_decode_page(_tokens_first(s[p], c), c["fmt"], torch.float32)[table].view(b, m * BS, hkv, d).transpose(1, 2)
            for p in ("k_pool", "v_pool"))
    there = torch.arange(m * BS, device="cuda")[None, :] < s["lens"][:, None]
    q = s["q"].float().view(b, hkv, hq // hkv, d)
    return _attend_plain(q, k, v, there[:, None, None], s["scale"]).view(b, hq, d).to(s["q"].dtype)


def _plain_cross(s):
    c = s["case"]
    hq, hkv, d, b = c["hq"], c["hkv"], c["d"], c["batch"]
    g = hq // hkv
    t_at = s["q_starts"][:-1, None] + torch.arange(c["t_hi"], device="cuda")
    t_ok = t_at < s["q_starts"][1:, None]
    n_at = torch.arange(c["n_hi"], device="cuda")[None, :]
    n_ok = n_at < s["k_lens"][:, None]
    n_at = torch.where(n_ok, s["k_starts"][:, None] + n_at, 0).long()
    q = s["q"].float()[torch.where(t_ok, t_at, 0).long()]  # padded to the longest target
    q = q.view(b, c["t_hi"], hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, c["t_hi"] * g, d)
    k, v = (s[x].float()[n_at].transpose(1, 2) for x in "kv")
    o = _attend_plain(q, k, v, n_ok[:, None, None], s["scale"])
    o = o.view(b, hkv, c["t_hi"], g, d).permute(0, 2, 1, 3, 4).reshape(b, c["t_hi"], hq, d)
    return o[t_ok].to(s["q"].dtype)


def _plain_rope(s):
    c = s["case"]
    half = c["rot"] // 2
    cs = s["cos_sin"][s["pos"]][:, None]
    cos, sin = cs[..., :half], cs[..., half:]

    def turned(x):
        x = x.float()
        r = x[..., :c["rot"]]
        a, b = (r[..., :half], r[..., half:]) if c["neox"] else (r[..., 0::2], r[..., 1::2])
        y = (a * cos - b * sin, b * cos + a * sin)
        y = torch.cat(y, -1) if c["neox"] else torch.stack(y, -1).flatten(-2)
        return torch.cat([y, x[..., c["rot"]:]], -1).to(s["q"].dtype)

    s["q_out"].copy_(turned(s["q"]))
    for pool, rows in ((s["k_pool"], turned(s["k"])), (s["v_pool"], s["v"])):
        tokens = pool if c["layout"] == "nhd" else pool.transpose(1, 2)
        tokens[s["slots"] // BS, s["slots"] % BS] = rows
    return s["q_out"], s["k_pool"], s["v_pool"]


# ------------------------------------------------------------------ what it costs, and what it should give

def work(case):
    c = case
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    if c["kind"] == "rope":
        t = c["tokens"]
        return {"bytes": t * (4.0 * (hq + 2 * hkv) * d + 4 * c["rot"] + 16), "flops": 3.0 * t * (hq + hkv) * c["rot"]}
    if c["kind"] == "cross":
        t, n = _cross_lens(c)
        return {"bytes": 4.0 * int(t.sum()) * hq * d + 4.0 * int(n.sum()) * hkv * d + 12 * len(t),
                "flops": 4.0 * hq * d * float((t * n).sum())}
    rows, shared, lens = _prefix_lens(c)
    once = float(_groups(c)[1].sum()) + float((lens - shared).sum())  # keys to read
    pages = once / BS
    return {"bytes": 4.0 * len(lens) * hq * d + 2 * once * hkv * _entry_bytes(c["fmt"], d) + 4 * pages + 4 * len(lens),
            "flops": 4.0 * hq * d * float(lens.sum())}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    return {"prefix": _exact_prefix, "cross": _exact_cross, "rope": _exact_rope}[c["kind"]](c, s)


def _softmax_rows(q, k, v, scale):
    """q [t][hq][d], k, v [n][hkv][d], all in 64 bits: every row over every key."""
    g = q.shape[1] // k.shape[1]
    out = torch.empty_like(q)
    for h in range(q.shape[1]):
        out[:, h] = torch.softmax(q[:, h] @ k[:, h // g].t() * scale, -1) @ v[:, h // g]
    return out


def _exact_prefix(c, s):
    q = s["q"].double()
    out = torch.empty_like(q)
    pools = [_tokens_first(s[p], c) for p in ("k_pool", "v_pool")]
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["bt"][b, :(n + BS - 1) // BS].long()
        k, v = (_decode_page(p[pages].flatten(0, 1)[:n], c["fmt"], torch.float64) for p in pools)
        out[b:b + 1] = _softmax_rows(q[b:b + 1], k, v, s["scale"])
    return out


def _exact_cross(c, s):
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    out = torch.empty_like(q)
    starts, lens = s["k_starts"].tolist(), s["k_lens"].tolist()
    edges = s["q_starts"].tolist()
    for b in range(len(lens)):
        at = slice(starts[b], starts[b] + lens[b])
        out[edges[b]:edges[b + 1]] = _softmax_rows(q[edges[b]:edges[b + 1]], k[at], v[at], s["scale"])
    return out


def _exact_rope(c, s):
    half, table = c["rot"] // 2, s["cos_sin"].double()
    turn = torch.complex(table[:, :half], table[:, half:])[s["pos"]][:, None]

    def turned(x):
        x = x.double().clone()
        r = x[..., :c["rot"]]
        pairs = r.view(*r.shape[:-1], 2, half).transpose(-1, -2) if c["neox"] else r.view(*r.shape[:-1], half, 2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        x[..., :c["rot"]] = (z.transpose(-1, -2) if c["neox"] else z).flatten(-2)
        return x

    pools = []
    for rows in (turned(s["k"]), s["v"].double()):
        n = s["k_pool"].shape[0] * BS
        pool = torch.zeros((n, *rows.shape[1:]), dtype=torch.float64, device="cuda")
        pool[s["slots"]] = rows
        pool = pool.view(-1, BS, *rows.shape[1:])
        pools.append(pool if c["layout"] == "nhd" else pool.transpose(1, 2).contiguous())
    return (turned(s["q"]), *pools)
