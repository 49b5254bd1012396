"""vmc_paged_attention_shared_prefix against 64 bits: a row's first shared tokens
come through the table row of its group's first row, the others through its own.
Every slot that no row attends holds 0xff bytes (NaNs)."""
import numpy as np
import pytest

from attn64 import attend, check

pytestmark = pytest.mark.gpu

F16, BF16, Q8, Q4 = 0, 1, 2, 3
# (format, q type): pages of the query's type, of the other one, GGUF with either
TYPES = [(F16, "f16"), (BF16, "bf16"), (F16, "bf16"), (BF16, "f16"), (Q8, "f16"), (Q8, "bf16"), (Q4, "f16"), (Q4, "bf16")]


def pool_values(raw, fmt, n, hkv, d):
    """Pool bytes [n entries][hkv] -> float64 values."""
    raw = raw.reshape(n, hkv, -1)
    if fmt in (F16, BF16):
        u = raw.view(np.uint16)
        if fmt == F16:
            return u.view(np.float16).astype(np.float64)
        return (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    b = raw.reshape(n, hkv, d // 32, -1)
    s = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    if fmt == Q8:
        q = b[..., 2:].view(np.int8).astype(np.float64)
    else:
        q = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8
    with np.errstate(invalid="ignore"):
        return (q * s).reshape(n, hkv, d)


class Batch:
    """Rows of `lens` tokens, groups [(rows, shared)] after `lead` rows of no group;
    every row has pages of its own for all its tokens (those that the group's first
    row stands for are never read), holes: (row, page) entries set to -1."""

    def __init__(self, dev, lens, groups, heads, d, fmt, qt, hnd=False, bs=16, seed=0, lead=0, holes=(), edit=None,
                 scale=None):
        import torch
        from vm_c_amd import capi
        self.capi, self.torch, self.dev = capi, torch, dev
        self.hq, self.hkv = heads
        self.d, self.fmt, self.qt, self.bs, self.hnd = d, fmt, qt, bs, hnd
        self.lens = np.asarray(lens, np.int64)
        rng = np.random.default_rng(seed)
        rows = len(self.lens)
        starts = np.concatenate([[0], np.cumsum([g[0] for g in groups])]).astype(np.int64) + lead
        self.shared, self.first = np.zeros(rows, np.int64), np.arange(rows)
        reach = np.maximum(self.lens, 0)
        for j, (n, s) in enumerate(groups):
            at = slice(starts[j], starts[j + 1])
            self.shared[at], self.first[at] = s, starts[j]
            if n:
                reach[starts[j]] = max(reach[starts[j]], s)  # the first row's table lists the shared pages
        pages = (reach + bs - 1) // bs
        nblk = int(pages.sum()) + 3
        perm = rng.permutation(nblk)
        bt = np.full((rows, max(1, int(pages.max(initial=0)))), -1, np.int32)
        at = 0
        for b in range(rows):
            bt[b, :pages[b]] = perm[at:at + pages[b]]
            at += pages[b]
        for r, p in holes:
            bt[r, p] = -1
        self.bt = bt
        dt = {"f16": torch.float16, "bf16": torch.bfloat16}
        self.dt = dt[qt]
        src = dt[{F16: "f16", BF16: "bf16"}.get(fmt, "f16")]
        n = nblk * bs
        k, v = (rng.standard_normal((n, self.hkv, d)).astype(np.float32) for _ in range(2))
        if edit:
            edit(self, k, v)
        layout = capi.LAYOUT_HND if hnd else capi.LAYOUT_NHD
        e = capi.kv_entry_bytes(fmt, d)
        kc, vc = (torch.full((n * self.hkv * e,), 0xff, dtype=torch.uint8, device=dev) for _ in range(2))
        used = np.unique(np.concatenate([self.slots(b) for b in range(rows)] + [np.zeros(0, np.int64)]))
        slots = np.where(np.isin(np.arange(n), used), np.arange(n), -1)
        capi.reshape_and_cache(torch.from_numpy(k).to(dev).to(src), torch.from_numpy(v).to(dev).to(src), kc, vc,
                               torch.from_numpy(slots).to(dev), bs, kv_format=fmt, layout=layout)
        self.kc, self.vc = kc, vc
        q = torch.from_numpy(rng.standard_normal((rows, self.hq, d)).astype(np.float32)).to(self.dt)
        self.q = q.to(dev)
        self.scale = d ** -0.5 if scale is None else scale
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
        self.t_bt, self.t_lens, self.t_starts = t(bt), t(self.lens), t(starts)
        self.t_shared = t([g[1] for g in groups])
        self.kw = dict(block_size=bs, kv_format=fmt, layout=layout)

    def slots(self, b):
        """Slots of row b's keys, holes left out."""
        p = np.arange(max(0, self.lens[b]))
        pg = self.bt[np.where(p < self.shared[b], self.first[b], b), p // self.bs].astype(np.int64)
        return (pg * self.bs + p % self.bs)[pg >= 0]

    def run(self, out=None, workspace=None, stream=None, q=None):
        q = self.q if q is None else q
        out = self.torch.full_like(q, float("nan")) if out is None else out
        return self.capi.paged_attention_shared_prefix(out, q, self.kc, self.vc, self.t_bt, self.t_lens, self.t_starts,
                                                       self.t_shared, self.hkv, self.scale, workspace=workspace,
                                                       stream=stream, **self.kw)

    def want(self, rows=None):
        raw = [x.cpu().numpy() for x in (self.kc, self.vc)]
        n = len(raw[0]) // (self.hkv * self.capi.kv_entry_bytes(self.fmt, self.d))
        if self.hnd:
            raw = [x.reshape(n // self.bs, self.hkv, self.bs, -1).swapaxes(1, 2).copy() for x in raw]
        k, v = (pool_values(x, self.fmt, n, self.hkv, self.d) for x in raw)
        q = self.q.cpu().double().numpy()
        # GGUF values may enter the products rounded to fp16
        e = 2.0 ** -11 if self.fmt in (Q8, Q4) else 0.0
        o, err = np.zeros(q.shape), np.zeros(q.shape)
        for b in range(len(q)) if rows is None else rows:
            at = self.slots(b)
            for h in range(self.hq):
                g = h // (self.hq // self.hkv)
                o[b, h], err[b, h] = attend(q[b, h], k[at, g], v[at, g], self.scale, self.qt, e, e)
        return o, err

    def check(self, got=None, rows=None, what=""):
        got = self.run() if got is None else got
        o, err = self.want(rows)
        got = got.cpu().double().numpy()
        at = slice(None) if rows is None else list(rows)
        check(got[at], o[at], err[at], what)
        return got


# lengths around pages and tiles, empty rows, rows shorter than what their group
# shares, prefixes that end inside a page, a group of one, one that shares nothing
LENS = [5, 40, 41, 300, 0, 16, 129, 200, 1, 64, 17, 130, 700, 33]
GROUPS = [(3, 40), (1, 250), (4, 128), (2, 0), (0, 9), (3, 17)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fmt,qt", TYPES)
@pytest.mark.parametrize("hnd", [False, True])
def test_formats(dev, d, fmt, qt, hnd):
    b = Batch(dev, LENS, GROUPS, (8, 2), d, fmt, qt, hnd, seed=d + fmt)
    got = b.check()
    assert (got[4] == 0).all()


# one row block and several of a wide group, groups of heads of 1 to 20, KV head
# counts that are no power of two
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", [(1, 1), (14, 2), (3, 3), (16, 1), (40, 2), (20, 10)])
def test_heads(dev, d, heads):
    b = Batch(dev, [70 + 3 * i for i in range(21)], [(17, 65), (3, 31)], heads, d, BF16, "bf16", seed=3)
    b.check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fmt", [F16, Q8])
@pytest.mark.parametrize("bs", [1, 8, 32, 48])
def test_block_sizes(dev, d, fmt, bs):
    Batch(dev, LENS, GROUPS, (8, 2), d, fmt, "f16", bs=bs, seed=bs).check()


# holes in shared and own pages, a row whose every page is one; a shared prefix that is
# nothing but holes
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fmt,qt", [(F16, "f16"), (Q4, "bf16")])
def test_holes(dev, d, fmt, qt):
    holes = [(0, 1), (3, 0), (5, 0), (7, 9), (12, 20), (13, 0), (13, 1), (13, 2)]
    Batch(dev, LENS, GROUPS, (8, 2), d, fmt, qt, seed=5, holes=holes).check()
    b = Batch(dev, [33, 32, 40, 12], [(4, 32)], (8, 2), d, fmt, qt, seed=6, holes=[(0, 0), (0, 1)])
    got = b.check()
    assert (got[1] == 0).all() and (got[3] == 0).all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_token_and_negative_scale(dev, d):
    Batch(dev, [1], [(1, 1)], (8, 2), d, F16, "f16").check()
    Batch(dev, [1, 1], [(2, 1)], (8, 2), d, BF16, "bf16").check()
    Batch(dev, LENS, GROUPS, (8, 2), d, BF16, "bf16", scale=-0.3).check()
    Batch(dev, LENS, GROUPS, (8, 2), d, F16, "f16", scale=0.0).check()


# rows before the first group, no group at all
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_of_no_group(dev, d):
    Batch(dev, LENS, [(4, 100)], (8, 2), d, F16, "f16", lead=5).check()
    b = Batch(dev, LENS, [], (8, 2), d, BF16, "bf16")
    b.check()
    out = b.torch.full_like(b.q, float("nan"))
    b.capi.paged_attention_shared_prefix(out, b.q, b.kc, b.vc, b.t_bt, b.t_lens, None, None, b.hkv, b.scale, **b.kw)
    b.check(out)


# a long prefix under many rows: several row blocks, ranges cut in the prefix and in
# the rows' own pages
@pytest.mark.parametrize("d,heads", [(64, (14, 2)), (128, (32, 8)), (256, (16, 2))])
@pytest.mark.parametrize("fmt,qt", [(F16, "f16"), (BF16, "bf16"), (Q8, "bf16"), (Q4, "f16")])
def test_long_prefix(dev, d, heads, fmt, qt):
    rng = np.random.default_rng(d)
    lens = np.concatenate([5000 + rng.integers(1, 900, 45), 700 + rng.integers(1, 3000, 5), rng.integers(1, 2000, 3)])
    b = Batch(dev, lens, [(45, 5000), (5, 700), (3, 0)], heads, d, fmt, qt, seed=8)
    b.check(rows=[0, 7, 31, 32, 44, 45, 49, 50, 52])


# the result does not depend on how the batch is grouped where the tables agree
@pytest.mark.parametrize("d", [64, 128, 256])
def test_same_as_plain_decode(dev, d):
    import torch
    b = Batch(dev, [400 + 7 * i for i in range(12)], [(12, 320)], (8, 2), d, F16, "f16", seed=2)
    got = b.check()
    bt = b.bt.copy()
    bt[:, :20] = bt[0, :20]
    out = torch.empty_like(b.q)
    b.capi.paged_attention_decode(out, b.q, b.kc, b.vc, torch.from_numpy(bt).to(dev), b.t_lens, 2, b.scale,
                                  kv_format=F16)
    o, err = b.want()
    check(out.cpu().double().numpy(), o, 2 * err, "plain decode")
    assert got.shape == o.shape


# infinities and NaNs that a row attends stay in that row
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fmt,qt", [(F16, "f16"), (BF16, "bf16")])
def test_values_not_finite(dev, d, fmt, qt):
    def edit(b, k, v):
        v[b.slots(2)[45], 0, 3] = np.inf    # an own key of row 2
        v[b.slots(4)[7], 1, 5] = -np.inf    # a shared key of rows 4 and 5
        k[b.slots(9)[1], 1, 0] = np.nan     # a key of row 9
    lens = [60, 70, 80, 90, 50, 60, 10, 20, 30, 40]
    b = Batch(dev, lens, [(4, 40), (2, 33)], (8, 2), d, fmt, qt, seed=4, edit=edit)
    got = b.run().cpu().double().numpy()
    o, err = b.want()
    odd = np.zeros(o.shape, bool)
    odd[2, :4, 3] = odd[4:6, 4:, 5] = odd[9, 4:] = True
    assert np.isposinf(got[2, :4, 3]).all() and np.isneginf(got[4:6, 4:, 5]).all() and np.isnan(got[9, 4:]).all()
    check(got[~odd], o[~odd], err[~odd])


# scores far apart: weights that underflow, and a prefix whose keys all weigh nothing
# against a row's own (and the other way round)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scores_far_apart(dev, d):
    def edit(b, k, v):
        k[b.slots(0)[5]] *= 30
        k[b.slots(1)[100]] *= 30
    b = Batch(dev, [90, 120, 200, 64], [(4, 64)], (8, 2), d, F16, "f16", seed=7, edit=edit, scale=1.0)
    b.check()


# more rows, and more groups, than the plan holds in LDS
@pytest.mark.parametrize("d", [64, 256])
def test_a_thousand_rows(dev, d):
    rng = np.random.default_rng(d)
    lens = rng.integers(0, 60, 1300)
    groups = [(int(n), int(s)) for n, s in zip(rng.integers(0, 4, 600), rng.integers(0, 50, 600))]
    while sum(g[0] for g in groups) > 1290:
        groups.pop()
    lens[5] = 4000
    Batch(dev, lens, groups, (4, 2), d, F16, "f16", seed=12, lead=7).check()
