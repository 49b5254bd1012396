"""Decode steps of an encoder-decoder layer, as a model runs them: rotation and append
(vmc_rope_and_cache), shared-prefix self attention over the pages, cross attention
over the encoder's states.  Eagerly, on streams, as replayed graphs, and over
memory past 32-bit offsets."""
import numpy as np
import pytest

from attn64 import attend, check
from test_gpu_cross_attention import Cross
from test_gpu_shared_prefix import BF16, F16, Q4, Q8, Batch, pool_values

pytestmark = pytest.mark.gpu
BS = 16


class Layer:
    """Rows of groups [(rows, shared tokens)], `own` tokens of each row behind them, room
    for `steps` more; encoder states of every group."""

    def __init__(self, dev, groups, own, heads, d, fmt, qt, steps, seed=0):
        import torch
        from vm_c_amd import capi
        self.capi, self.torch, self.dev = capi, torch, dev
        self.hq, self.hkv, self.d, self.fmt, self.qt = *heads, d, fmt, qt
        rng = np.random.default_rng(seed)
        self.rng = rng
        self.dt = {"f16": torch.float16, "bf16": torch.bfloat16}[qt]
        rows = sum(g[0] for g in groups)
        self.starts = np.concatenate([[0], np.cumsum([g[0] for g in groups])])
        self.shared = np.repeat([g[1] for g in groups], [g[0] for g in groups])
        self.lens = self.shared + np.asarray(own)
        # whole shared pages are one for the group; a row's other pages are its own
        mb = int((self.lens + steps + BS - 1).max() // BS + 1)
        self.bt = np.full((rows, mb), -1, np.int32)
        nblk = int(sum((n + steps + BS - 1) // BS for n in self.lens)) + 2
        free = list(rng.permutation(nblk))
        self.share = np.zeros(len(groups), np.int64)
        for j, (n, s) in enumerate(groups):
            self.share[j] = s // BS * BS
            common = [free.pop() for _ in range(s // BS)]
            for r in range(self.starts[j], self.starts[j + 1]):
                more = (self.lens[r] + steps + BS - 1) // BS - len(common)
                self.bt[r, :len(common) + more] = common + [free.pop() for _ in range(more)]
        self.nblk = nblk
        e = capi.kv_entry_bytes(fmt, d)
        self.kc, self.vc = (torch.full((nblk * BS * self.hkv * e,), 0xff, dtype=torch.uint8, device=dev) for _ in range(2))
        slots = np.unique(np.concatenate([self.slots(r) for r in range(rows)]))
        src = {F16: torch.float16, BF16: torch.bfloat16}.get(fmt, torch.float16)
        kv = torch.from_numpy(rng.standard_normal((2, len(slots), self.hkv, d)).astype(np.float32)).to(dev).to(src)
        capi.reshape_and_cache(kv[0], kv[1], self.kc, self.vc, torch.from_numpy(slots).to(dev), BS, kv_format=fmt)
        half = d // 2
        ang = torch.arange(int(self.lens.max()) + steps + 1, dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(half) / half)
        self.table = torch.cat([ang.cos(), ang.sin()], 1).float().to(dev)
        n = rng.integers(20, 200, len(groups))
        self.k_lens, self.k_starts = n, np.concatenate([[0], np.cumsum(n)[:-1]])
        self.enc = torch.from_numpy(rng.standard_normal((int(n.sum()), 2, self.hkv, d)).astype(np.float32)).to(dev).to(self.dt)
        i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
        self.t_bt, self.t_starts, self.t_share = i32(self.bt), i32(self.starts), i32(self.share)
        self.t_ks, self.t_kl = i32(self.k_starts), i32(self.k_lens)
        self.t_lens = i32(self.lens)
        self.t_pos = torch.zeros(rows, dtype=torch.int64, device=dev)
        self.t_slots = torch.zeros(rows, dtype=torch.int64, device=dev)
        self.qkv = torch.zeros((rows, self.hq + 2 * self.hkv, d), dtype=self.dt, device=dev)
        shape = (rows, self.hq, d)
        self.q, self.a, self.x = (torch.zeros(shape, dtype=self.dt, device=dev) for _ in range(3))
        self.ws = [torch.empty(max(1, n), dtype=torch.uint8, device=dev) for n in (
            capi.shared_prefix_workspace_size(rows, self.hq, self.hkv, d, len(groups)),
            capi.cross_attention_workspace_size(rows, len(groups), self.hq, self.hkv, d))]
        self.scale = d ** -0.5

    def slots(self, r):
        p = np.arange(self.lens[r])
        return self.bt[r, p // BS].astype(np.int64) * BS + p % BS

    def step(self):
        """One more token of every row: the step's tensors, in place."""
        t = self.torch
        pos = self.lens.copy()
        self.lens = self.lens + 1
        slot = self.bt[np.arange(len(pos)), pos // BS].astype(np.int64) * BS + pos % BS
        self.t_pos.copy_(t.from_numpy(pos.astype(np.int64)))
        self.t_slots.copy_(t.from_numpy(slot))
        self.t_lens.copy_(t.from_numpy(self.lens.astype(np.int32)))
        self.qkv.copy_(t.from_numpy(self.rng.standard_normal(tuple(self.qkv.shape)).astype(np.float32)).to(self.dt))

    def run(self, stream=None):
        h, k = self.hq, self.hkv
        kw = dict(kv_format=self.fmt, stream=stream)
        self.capi.rope_and_cache(self.qkv[:, :h], self.qkv[:, h:h + k], self.qkv[:, h + k:], self.table, self.t_pos,
                                 self.kc, self.vc, self.t_slots, BS, query_out=self.q, **kw)
        self.capi.paged_attention_shared_prefix(self.a, self.q, self.kc, self.vc, self.t_bt, self.t_lens, self.t_starts,
                                                self.t_share, k, self.scale, workspace=self.ws[0], **kw)
        self.capi.cross_attention(self.x, self.a, self.enc[:, 0], self.enc[:, 1], self.t_starts, self.t_ks, self.t_kl,
                                  self.scale, workspace=self.ws[1], stream=stream)

    def outputs(self):
        return [t.clone() for t in (self.q, self.a, self.x, self.kc, self.vc)]

    def check(self):
        raw = [c.cpu().numpy() for c in (self.kc, self.vc)]
        pk, pv = (pool_values(c, self.fmt, self.nblk * BS, self.hkv, self.d) for c in raw)
        q, a, x = (t.cpu().double().numpy() for t in (self.q, self.a, self.x))
        enc = self.enc.cpu().double().numpy()
        e = 2.0 ** -11 if self.fmt in (Q8, Q4) else 0.0
        for r in range(len(q)):
            s, j = self.slots(r), int(np.searchsorted(self.starts, r, "right")) - 1
            at = slice(self.k_starts[j], self.k_starts[j] + self.k_lens[j])
            for h in range(self.hq):
                g = h // (self.hq // self.hkv)
                check(a[r, h], *attend(q[r, h], pk[s, g], pv[s, g], self.scale, self.qt, e, e), what=f"self {r} {h}")
                check(x[r, h], *attend(a[r, h], enc[at, 0, g], enc[at, 1, g], self.scale, self.qt), what=f"cross {r} {h}")


GROUPS, OWN = [(5, 200), (1, 0), (3, 70)], [1, 30, 16, 15, 7, 40, 3, 100, 33]


@pytest.mark.parametrize("d,heads", [(64, (6, 2)), (128, (8, 2)), (256, (4, 1))])
@pytest.mark.parametrize("fmt,qt", [(F16, "f16"), (BF16, "bf16"), (Q8, "f16"), (Q4, "bf16")])
def test_steps(dev, d, heads, fmt, qt):
    m = Layer(dev, GROUPS, OWN, heads, d, fmt, qt, steps=20, seed=d)
    for i in range(20):  # rows pass page ends and tile ends
        m.step()
        m.run()
        if i in (0, 9, 19):
            m.check()


@pytest.mark.parametrize("d,heads,fmt,qt", [(64, (6, 2), F16, "f16"), (128, (8, 2), Q8, "bf16"), (128, (8, 2), BF16, "bf16"),
                                            (256, (4, 1), BF16, "bf16")])
def test_replayed_graph(dev, d, heads, fmt, qt):
    import torch
    m = Layer(dev, GROUPS, OWN, heads, d, fmt, qt, steps=20, seed=d)
    twin = Layer(dev, GROUPS, OWN, heads, d, fmt, qt, steps=20, seed=d)
    for x in (m, twin):
        x.step()
        x.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.run()
    for i in range(6):
        m.step()
        g.replay()
        twin.step()
        twin.run()  # eager work of its own between the replays
        for a, b in zip(m.outputs(), twin.outputs()):
            assert torch.equal(a, b), i
        if i % 2:
            torch.cuda.synchronize()
    # other groups, in the arrays that the graph reads
    for x in (m, twin):
        x.t_share.zero_()
        x.step()
    g.replay()
    twin.run()
    assert all(torch.equal(a, b) for a, b in zip(m.outputs(), twin.outputs()))
    m.check()


def test_two_streams_at_once(dev):
    """Two layers on streams of their own, each with its workspaces, against one after the
    other on the current stream."""
    import torch
    kinds = [((8, 2), 128, BF16, "bf16"), ((6, 2), 64, F16, "f16")]
    ms = [Layer(dev, GROUPS, OWN, h, d, f, t, steps=12, seed=3) for h, d, f, t in kinds]
    twins = [Layer(dev, GROUPS, OWN, h, d, f, t, steps=12, seed=3) for h, d, f, t in kinds]
    streams = [torch.cuda.Stream() for _ in ms]
    for _ in range(10):
        for m, s in zip(ms, streams):
            m.step()
            s.wait_stream(torch.cuda.current_stream())
            m.run(stream=s)
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for m, t in zip(ms, twins):
            t.step()
            t.run()
            assert all(torch.equal(a, b) for a, b in zip(m.outputs(), t.outputs()))


def test_workspace_sizes(dev):
    """A workspace of one byte less is refused, one of the size asked for is enough, also
    where it held another call's values or NaNs."""
    import torch
    b = Batch(dev, [100, 300, 7], [(2, 64), (1, 0)], (8, 2), 128, F16, "f16")
    n = b.capi.shared_prefix_workspace_size(3, 8, 2, 128, 2)
    ws = torch.full((n,), 0xff, dtype=torch.uint8, device=dev)
    with pytest.raises(b.capi.VmcError):
        b.run(workspace=ws[:-1])
    o, err = b.want()
    for _ in range(2):
        check(b.run(workspace=ws).cpu().double().numpy(), o, err)
    c = Cross(dev, [3, 100], [70, 500], (8, 2), 128, "bf16")
    n = b.capi.cross_attention_workspace_size(103, 2, 8, 2, 128)
    ws = torch.full((n,), 0xff, dtype=torch.uint8, device=dev)
    with pytest.raises(b.capi.VmcError):
        c.run(workspace=ws[:-1])
    for _ in range(2):
        c.check(c.run(workspace=ws))


# pools of more than 2^32 bytes, pages at their end
@pytest.mark.parametrize("fmt,qt", [(BF16, "bf16"), (Q8, "f16")])
def test_pages_past_32_bits(dev, fmt, qt):
    import torch
    from vm_c_amd import capi
    d, hq, hkv = 256, 16, 8
    e = capi.kv_entry_bytes(fmt, d)
    page = BS * hkv * e
    nblk = (1 << 32) // page + 64
    lens, shared = np.array([200, 150, 97]), 80
    need = (lens + BS - 1) // BS
    bt = np.full((3, int(need.max())), -1, np.int32)
    used = iter(range(nblk - int(need.sum()), nblk))
    for r in range(3):
        bt[r, :need[r]] = [next(used) for _ in range(need[r])]
    bt[1:, :shared // BS] = bt[0, :shared // BS]
    kc, vc = (torch.empty(nblk * page, dtype=torch.uint8, device=dev) for _ in range(2))
    table = torch.zeros((256, d), device=dev)
    table[:, :d // 2] = 1.0  # no turn
    rng = np.random.default_rng(5)
    dt = torch.bfloat16 if qt == "bf16" else torch.float16
    k, v = {}, {}
    for r in range(3):
        p = np.arange(lens[r])
        slots = bt[r, p // BS].astype(np.int64) * BS + p % BS
        x = torch.from_numpy(rng.standard_normal((lens[r], hq + 2 * hkv, d)).astype(np.float32)).to(dt).to(dev)
        if r:
            x[:shared, hq:] = first[:shared, hq:]
        else:
            first = x
        capi.rope_and_cache(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], table, torch.from_numpy(p).to(dev), kc, vc,
                            torch.from_numpy(slots).to(dev), BS, kv_format=fmt)
        idx = torch.from_numpy(slots).to(dev)
        k[r], v[r] = (pool_values(c.view(-1, hkv * e)[idx].cpu().numpy(), fmt, lens[r], hkv, d) for c in (kc, vc))
        if fmt == BF16:
            assert np.array_equal(k[r], x[:, hq:hq + hkv].cpu().double().numpy())
    q = torch.from_numpy(rng.standard_normal((3, hq, d)).astype(np.float32)).to(dt).to(dev)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    out = capi.paged_attention_shared_prefix(torch.empty_like(q), q, kc, vc, i32(bt), i32(lens), i32([0, 3]),
                                             i32([shared]), hkv, d ** -0.5, block_size=BS, kv_format=fmt)
    out, q = out.cpu().double().numpy(), q.cpu().double().numpy()
    ev = 2.0 ** -11 if fmt == Q8 else 0.0
    for r in range(3):
        for h in range(hq):
            g = h // (hq // hkv)
            check(out[r, h], *attend(q[r, h], k[r][:, g], v[r][:, g], d ** -0.5, qt, ev, ev), what=f"{r} {h}")


@pytest.mark.parametrize("d", [64, 128, 256])
def test_states_past_32_bits(dev, d):
    """Tokens of states 8 MB apart: 5.4 GB from the first to the last."""
    import torch
    from vm_c_amd import capi
    n, stride = 650, 1 << 22
    rng = np.random.default_rng(6)
    kv = torch.empty(n * stride, dtype=torch.bfloat16, device=dev).view(n, stride)
    x = torch.from_numpy(rng.standard_normal((n, 2, 2, d)).astype(np.float32)).to(torch.bfloat16).to(dev)
    kv[:, :4 * d] = x.view(n, 4 * d)
    k, v = (kv[:, i * 2 * d:(i + 1) * 2 * d].unflatten(1, (2, d)) for i in range(2))
    t = np.array([1, 40, 3])
    q = torch.from_numpy(rng.standard_normal((int(t.sum()), 4, d)).astype(np.float32)).to(torch.bfloat16).to(dev)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    edges, k0, kn = np.concatenate([[0], np.cumsum(t)]), np.array([0, 500, 600]), np.array([650, 150, 50])
    out = capi.cross_attention(torch.empty_like(q), q, k, v, i32(edges), i32(k0), i32(kn), d ** -0.5)
    out, q, x = out.cpu().double().numpy(), q.cpu().double().numpy(), x.cpu().double().numpy()
    for s in range(3):
        at = slice(k0[s], k0[s] + kn[s])
        for r in range(edges[s], edges[s + 1], 7):
            for h in range(4):
                check(out[r, h], *attend(q[r, h], x[at, 0, h // 2], x[at, 1, h // 2], d ** -0.5, "bf16"), what=f"{r} {h}")
