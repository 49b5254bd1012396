"""vmc_cross_attention against 64 bits: rows of a decoder over the states of their
sequence, any strides, no causal mask."""
import numpy as np
import pytest

from attn64 import attend, check

pytestmark = pytest.mark.gpu


class Cross:
    """t[s] rows over n[s] states of sequence s.  gap: rows of no sequence before,
    and behind; slack: states between the sequences (NaN)."""

    def __init__(self, dev, t, n, heads, d, qt, seed=0, gap=(0, 0), slack=0, fused=True, heads_first=False, scale=None,
                 edit=None, share=None):
        import torch
        from vm_c_amd import capi
        self.capi, self.torch = capi, torch
        self.hq, self.hkv = heads
        self.d, self.qt = d, qt
        dt = {"f16": torch.float16, "bf16": torch.bfloat16}[qt]
        rng = np.random.default_rng(seed)
        self.t_edges = np.concatenate([[0], np.cumsum(t)]) + gap[0]
        self.n = np.asarray(n)
        self.k0 = np.concatenate([[0], np.cumsum(self.n + slack)[:-1]]) if len(n) else np.zeros(0, np.int64)
        if share is not None:  # sequence s uses the states of sequence share[s]
            self.k0, self.n = self.k0[share], self.n[share]
        rows, keys = int(self.t_edges[-1]) + gap[1], int((np.asarray(n) + slack).sum())
        kv = rng.standard_normal((2, keys, self.hkv, d)).astype(np.float32)
        used = np.zeros(keys, bool)
        for k0, m in zip(self.k0, self.n):
            used[k0:k0 + m] = True
        kv[:, ~used] = np.nan
        if edit:
            edit(self, kv[0], kv[1])
        kv = torch.from_numpy(kv).to(dev).to(dt)
        if fused:  # [key][k, v][head][d]
            kv = kv.permute(1, 0, 2, 3).contiguous()
            self.k, self.v = kv[:, 0], kv[:, 1]
        elif heads_first:  # [head][key][d]
            self.k, self.v = (x.permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in kv)
        else:
            self.k, self.v = kv[0], kv[1]
        q = torch.from_numpy(rng.standard_normal((rows, self.hq + 1, d)).astype(np.float32)).to(dev).to(dt)
        self.q = q[:, :self.hq] if fused else q[:, :self.hq].contiguous()
        i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
        self.starts, self.k_starts, self.k_lens = i32(self.t_edges), i32(self.k0), i32(self.n)
        self.scale = d ** -0.5 if scale is None else scale

    def run(self, out=None, workspace=None, stream=None):
        if out is None:
            out = self.torch.full(self.q.shape, 7.0, dtype=self.q.dtype, device=self.q.device)
        return self.capi.cross_attention(out, self.q, self.k, self.v, self.starts, self.k_starts, self.k_lens,
                                         self.scale, workspace=workspace, stream=stream)

    def want(self, step=1, mixed=False):
        q, k, v = (x.cpu().double().numpy() for x in (self.q, self.k, self.v))
        o, err = np.full(q.shape, 7.0), np.zeros(q.shape)  # rows of no sequence stay
        seen = np.zeros(len(q), bool)
        seen[:self.t_edges[0]] = seen[self.t_edges[-1]:] = True
        for s in range(len(self.n)):
            at = slice(self.k0[s], self.k0[s] + self.n[s])
            for r in range(self.t_edges[s], self.t_edges[s + 1], 1):
                if (r - self.t_edges[s]) % step and r != self.t_edges[s + 1] - 1:
                    continue
                seen[r] = True
                for h in range(self.hq):
                    g = h // (self.hq // self.hkv)
                    o[r, h], err[r, h] = attend(q[r, h], k[at, g], v[at, g], self.scale, self.qt,
                                                  mixed=mixed)
        return o, err, seen

    def check(self, got=None, step=1, mixed=False):
        got = (self.run() if got is None else got).cpu().double().numpy()
        o, err, seen = self.want(step, mixed)
        check(got[seen], o[seen], err[seen])
        return got


T = [1, 0, 7, 33, 2, 1, 130, 5]
N = [1, 40, 64, 65, 0, 500, 31, 129]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("qt", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["fused", "plain", "heads first"])
def test_ragged(dev, d, qt, layout):
    c = Cross(dev, T, N, (8, 2), d, qt, seed=d, gap=(2, 3), slack=5, fused=layout == "fused",
              heads_first=layout == "heads first")
    got = c.check()
    assert (got[c.t_edges[4]:c.t_edges[5]] == 0).all()  # no states


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", [(1, 1), (14, 2), (10, 10), (16, 1), (40, 2)])
@pytest.mark.parametrize("t", [1, 5, 70])
def test_heads(dev, d, heads, t):
    Cross(dev, [t, t, 1], [100, 65, 17], heads, d, "bf16", seed=t).check()


# single tokens over long states: keys cut into many pieces
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("qt", ["f16", "bf16"])
@pytest.mark.parametrize("t", [1, 4])
def test_few_rows_long_states(dev, d, qt, t):
    Cross(dev, [t] * 3, [9001, 1500, 4097], (8, 4), d, qt, seed=t).check()


# whole targets: several row blocks a sequence
@pytest.mark.parametrize("d,heads", [(64, (12, 12)), (128, (32, 8)), (256, (16, 2))])
@pytest.mark.parametrize("qt", ["f16", "bf16"])
def test_long_targets(dev, d, heads, qt):
    Cross(dev, [700, 333, 64], [1111, 64, 1500], heads, d, qt, seed=2).check(step=37)


# the hypotheses of one input share its states
@pytest.mark.parametrize("d", [64, 128, 256])
def test_shared_states(dev, d):
    Cross(dev, [1, 1, 4, 1], [300, 77, 5, 64], (8, 2), d, "f16", seed=3, share=[0, 0, 1, 0]).check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_scales(dev, d):
    for scale in (-0.2, 0.0, 1.0):
        Cross(dev, [1, 40], [200, 130], (8, 2), d, "f16", seed=4, scale=scale).check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_short_sequences(dev, d):
    rng = np.random.default_rng(d)
    Cross(dev, rng.integers(0, 4, 300), rng.integers(0, 40, 300), (8, 2), d, "bf16", seed=5, gap=(0, 9)).check()


# infinities and NaNs of one sequence's states stay in its rows; keys ranges that reach
# past the states are cut
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [1, 40])
def test_values_not_finite(dev, d, t):
    def edit(c, k, v):
        v[c.k0[1] + 3, 0, 2] = np.inf
        k[c.k0[2] + 1, 1, 0] = np.nan
    c = Cross(dev, [t, t, t], [70, 70, 70], (8, 2), d, "bf16", seed=6, edit=edit)
    got = c.run().cpu().double().numpy()
    o, err, _ = c.want()
    odd = np.zeros(o.shape, bool)
    odd[t:2 * t, :4, 2] = odd[2 * t:, 4:] = True
    assert np.isposinf(got[t:2 * t, :4, 2]).all() and np.isnan(got[2 * t:, 4:]).all()
    check(got[~odd], o[~odd], err[~odd])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [1, 40])
def test_ranges_are_cut(dev, d, t):
    c = Cross(dev, [t, t, t], [70, 70, 70], (8, 2), d, "f16", seed=7)
    c.k_starts.copy_(c.torch.tensor([-5, 200, 300]))
    c.k_lens.copy_(c.torch.tensor([20, 100, 9]))
    c.k0, c.n = np.array([0, 200, 0]), np.array([15, 10, 0])
    c.check()


# so many items that each workgroup takes whole ones: sequences without rows or without
# states, padding rows, a row block cut in the middle
@pytest.mark.parametrize("d,heads", [(64, (32, 8)), (128, (32, 8)), (256, (16, 16))])
@pytest.mark.parametrize("qt", ["f16", "bf16"])
def test_whole_items(dev, d, heads, qt):
    rng = np.random.default_rng(d)
    n_seq = 130
    t = rng.integers(30, 40, n_seq) if heads[0] > heads[1] else rng.integers(130, 150, n_seq)
    n = rng.integers(1, 200, n_seq)
    t[3], n[7] = 0, 0
    t[40] = 1100
    c = Cross(dev, t, n, heads, d, qt, seed=9, gap=(4, 5))
    got = c.check(step=97)
    assert (got[c.t_edges[7]:c.t_edges[8]] == 0).all()


# V of any magnitude: all values of a size, single outliers, one dim far from the others,
# chunks of 16 keys of different sizes, values that no 16-bit scale fits
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [3, 70])
@pytest.mark.parametrize("size", ["300", "7e4", "1e30", "1e-5", "1e-12", "1e-30", "outlier", "dim", "chunks", "zeros"])
def test_value_magnitudes(dev, d, t, size):
    def edit(c, k, v):
        if size == "outlier":
            v[77, 0, 5] = 3e4
            v[150, 1, 9] = 1e6
        elif size == "dim":
            v[..., 7] *= 1e-4
            v[..., 8] *= 1e3
        elif size == "chunks":
            v *= np.repeat([1, 1e-6, 700, 1e-3, 1, 9e4, 1e-9], 32)[:200, None, None]
        elif size == "zeros":
            v[16:80] = 0
            v[100:] = 0
        else:
            v *= float(size)
    Cross(dev, [t, t], [130, 70], (8, 2), d, "bf16", seed=10, edit=edit).check(mixed=True)


# more sequences than the plan holds in LDS
@pytest.mark.parametrize("d", [64, 256])
def test_a_thousand_sequences(dev, d):
    rng = np.random.default_rng(d)
    n = rng.integers(0, 20, 1500)
    n[700] = 3000
    Cross(dev, rng.integers(0, 3, 1500), n, (4, 2), d, "f16", seed=11, gap=(3, 2)).check()
