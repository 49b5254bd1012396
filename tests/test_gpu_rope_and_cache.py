"""vmc_rope_and_cache: Q and K rotated as 64 bits says, to one rounding of the fp32
result; pages byte for byte what vmc_reshape_and_cache writes of the rotated K."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BS = 16
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Rope:
    def __init__(self, dev, t, heads, d, rot, qt, seed=0, fused=True, max_pos=5000):
        import torch
        self.torch = torch
        self.hq, self.hkv, self.d, self.rot, self.qt = *heads, d, rot, qt
        self.dt = {"f16": torch.float16, "bf16": torch.bfloat16}[qt]
        g = torch.Generator().manual_seed(seed)
        x = torch.randn((t, self.hq + 2 * self.hkv + 1, d), generator=g).to(self.dt).to(dev)
        e = [0, self.hq, self.hq + self.hkv, self.hq + 2 * self.hkv]
        self.q, self.k, self.v = (x[:, a:b] if fused else x[:, a:b].contiguous() for a, b in zip(e, e[1:]))
        half = rot // 2
        ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half) / half)
        self.table = torch.cat([ang.cos(), ang.sin()], 1).float().to(dev)
        self.pos = torch.randint(0, max_pos, (t,), generator=g).to(dev)
        self.pages = (t + BS - 1) // BS + 1
        self.slots = torch.randperm(self.pages * BS, generator=g)[:t].to(dev)

    def want(self, x, neox):
        """float64 values and the allowed error."""
        x = x.double()
        half = self.rot // 2
        cs = self.table.double()[self.pos.clamp(0, len(self.table) - 1)][:, None]
        cos, sin = cs[..., :half], cs[..., half:]
        r = x[..., :self.rot]
        a, b = (r[..., :half], r[..., half:]) if neox else (r[..., 0::2], r[..., 1::2])
        join = (lambda u, w: self.torch.cat([u, w], -1)) if neox else \
            (lambda u, w: self.torch.stack([u, w], -1).flatten(-2))
        y = self.torch.cat([join(a * cos - b * sin, b * cos + a * sin), x[..., self.rot:]], -1)
        # two products and a sum in fp32, then one rounding to the type
        size = join((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs())
        err = self.torch.cat([size * 2.0 ** -23, self.torch.zeros_like(x[..., self.rot:])], -1)
        return y, err + self.torch.where(err > 0, (y.abs() + err) * HALF_STEP[self.qt] + 2.0 ** -25, 0.0)

    def pools(self, fmt):
        from vm_c_amd import capi
        n = self.pages * BS * self.hkv * capi.kv_entry_bytes(fmt, self.d)
        return [self.torch.full((n,), 0x5a, dtype=self.torch.uint8, device=self.q.device) for _ in range(2)]


def _close(got, want, err):
    bad = ~((got.double() - want).abs() <= err)
    assert not bad.any(), (int(bad.sum()), got[bad][0].item(), want[bad][0].item(), err[bad][0].item())


@pytest.mark.parametrize("d,rot", [(64, 64), (64, 16), (64, 32), (128, 128), (128, 64), (256, 256), (256, 64), (256, 48)])
@pytest.mark.parametrize("qt", ["f16", "bf16"])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("fmt", [0, 1, 2, 3])
@pytest.mark.parametrize("t,heads", [(1, (5, 1)), (37, (8, 2)), (70, (10, 5))])
def test_rotation_and_pages(dev, d, rot, qt, neox, fmt, t, heads):
    from vm_c_amd import capi
    for fused, layout in ((True, capi.LAYOUT_NHD), (False, capi.LAYOUT_HND)):
        r = Rope(dev, t, heads, d, rot, qt, seed=t + d, fused=fused)
        r.slots[t // 2] = -1
        (kc, vc), (kr, vr) = r.pools(fmt), r.pools(fmt)
        k_out = r.torch.empty((t, r.hkv, d), dtype=r.dt, device=dev)
        keep = [x.clone() for x in (r.q, r.k, r.v)]
        kw = dict(kv_format=fmt, layout=layout)
        out = capi.rope_and_cache(r.q, r.k, r.v, r.table, r.pos, kc, vc, r.slots, BS, key_out=k_out, is_neox=neox, **kw)
        _close(out, *r.want(r.q, neox))
        _close(k_out, *r.want(r.k, neox))
        assert r.torch.equal(out[..., rot:], r.q[..., rot:])
        capi.reshape_and_cache(k_out, r.v.contiguous(), kr, vr, r.slots, BS, **kw)
        assert r.torch.equal(kc, kr) and r.torch.equal(vc, vr)
        assert all(r.torch.equal(a, b) for a, b in zip(keep, (r.q, r.k, r.v)))  # the inputs stay


# without pages, without key_out, in place, pages with a stride
@pytest.mark.parametrize("d", [64, 128, 256])
def test_outputs(dev, d):
    from vm_c_amd import capi
    r = Rope(dev, 33, (8, 2), d, d, "bf16", fused=False)
    k_out = r.torch.empty_like(r.k)
    out = capi.rope_and_cache(r.q, r.k, None, r.table, r.pos, key_out=k_out)
    _close(out, *r.want(r.q, True))
    _close(k_out, *r.want(r.k, True))
    kc, vc = r.pools(1)
    stride = BS * r.hkv * 2 * d + 32
    kc2, vc2 = (r.torch.zeros(r.pages * stride, dtype=r.torch.uint8, device=dev) for _ in range(2))
    capi.rope_and_cache(r.q, r.k, r.v, r.table, r.pos, kc, vc, r.slots, BS, kv_format=1)
    capi.rope_and_cache(r.q, r.k, r.v, r.table, r.pos, kc2, vc2, r.slots, BS, kv_format=1, cache_stride=stride)
    page = lambda x, s: x.view(-1, s)[:, :BS * r.hkv * 2 * d]  # noqa: E731
    written = (r.slots // BS).unique()
    a, b = page(kc, stride - 32)[written], page(kc2, stride)[written]
    assert r.torch.equal(a[a != 0x5a], b[a != 0x5a])
    q, k = r.q.clone(), r.k.clone()
    capi.rope_and_cache(q, k, None, r.table, r.pos, query_out=q, key_out=k)
    assert r.torch.equal(q, out) and r.torch.equal(k, k_out)


# a position outside the table: the token is skipped
def test_padding_tokens(dev):
    from vm_c_amd import capi
    r = Rope(dev, 40, (8, 2), 128, 128, "f16", max_pos=300)
    kc, vc = r.pools(0)
    ref_k, ref_v = kc.clone(), vc.clone()
    ok = r.torch.ones(40, dtype=r.torch.bool, device=dev)
    out = capi.rope_and_cache(r.q, r.k, r.v, r.table, r.pos, ref_k, ref_v, r.slots.where(r.torch.arange(40, device=dev) % 3 != 0, -1), BS)
    bad = r.pos.clone()
    bad[0::6], bad[3::6] = -1, 300
    ok[0::3] = False
    got = r.torch.full_like(out, 9.0)
    capi.rope_and_cache(r.q, r.k, r.v, r.table, bad, kc, vc, r.slots, BS, query_out=got)
    assert r.torch.equal(got[ok], out[ok]) and (got[~ok] == 9.0).all()
    assert r.torch.equal(kc, ref_k) and r.torch.equal(vc, ref_v)


# a prefill step: many workgroups, an odd number of tokens
@pytest.mark.parametrize("d,heads,rot", [(64, (14, 2), 64), (128, (32, 8), 128), (256, (16, 2), 64)])
def test_large(dev, d, heads, rot):
    from vm_c_amd import capi
    r = Rope(dev, 3001, heads, d, rot, "bf16", seed=1)
    kc, vc = r.pools(1)
    kr, vr = r.pools(1)
    k_out = r.torch.empty((3001, r.hkv, d), dtype=r.dt, device=dev)
    out = capi.rope_and_cache(r.q, r.k, r.v, r.table, r.pos, kc, vc, r.slots, BS, key_out=k_out, kv_format=1)
    _close(out, *r.want(r.q, True))
    _close(k_out, *r.want(r.k, True))
    capi.reshape_and_cache(k_out, r.v.contiguous(), kr, vr, r.slots, BS, kv_format=1)
    assert r.torch.equal(kc, kr) and r.torch.equal(vc, vr)
