"""Arguments that the shared-prefix decode, the cross attention and the rotation
with append refuse before any launch."""
import ctypes as C

import pytest

P = C.c_void_p(4096)


def _prefix(lib, **kw):
    a = dict(out=P, q=P, k=P, v=P, bt=P, lens=P, starts=P, shared=P, batch=4, groups=2, hq=8, hkv=2, d=128, bs=16,
             blocks=64, scale=C.c_float(0.1), qt=0, fmt=0, layout=0, ws=P, ws_bytes=1 << 34, stream=None)
    a.update(kw)
    return lib.vmc_paged_attention_shared_prefix(*a.values())


def _cross(lib, **kw):
    a = dict(out=P, q=P, k=P, v=P, qs=P, ks=P, kl=P, t=4, n=100, s=2, hq=8, hkv=2, d=128, q_ts=1024, q_hs=128, k_ts=256,
             k_hs=128, v_ts=256, v_hs=128, scale=C.c_float(0.1), dt=0, ws=P, ws_bytes=1 << 34, stream=None)
    a.update(kw)
    return lib.vmc_cross_attention(*a.values())


def _rope(lib, **kw):
    a = dict(q_out=P, k_out=None, q=P, k=P, v=P, cs=P, pos=P, kc=P, vc=P, slots=P, t=4, hq=8, hkv=2, d=128, rot=128,
             max_pos=100, q_ts=1024, k_ts=256, v_ts=256, neox=1, bs=16, stride=0, fmt=0, layout=0, dt=0, stream=None)
    a.update(kw)
    return lib.vmc_rope_and_cache(*a.values())


PREFIX = [dict(batch=-1), dict(groups=-1), dict(hq=0), dict(hkv=0), dict(hkv=3), dict(d=96), dict(bs=0), dict(bs=-16),
          dict(blocks=-1), dict(blocks=1 << 28), dict(qt=2), dict(fmt=4), dict(fmt=-1), dict(layout=2), dict(out=None),
          dict(q=None), dict(k=None), dict(v=None), dict(bt=None), dict(lens=None), dict(starts=None),
          dict(shared=None), dict(k=C.c_void_p(4098)), dict(v=C.c_void_p(4097), fmt=2), dict(out=C.c_void_p(4097)),
          dict(batch=1 << 21)]
CROSS = [dict(t=-1), dict(n=-1), dict(s=-1), dict(hq=7), dict(d=80), dict(q_ts=127), dict(k_hs=64), dict(v_ts=257),
         dict(k_ts=-256), dict(dt=2), dict(out=None), dict(q=None), dict(k=None), dict(v=None), dict(qs=None),
         dict(ks=None), dict(kl=None), dict(k=C.c_void_p(4098)), dict(t=1 << 24), dict(t=1 << 23, hq=256)]
ROPE = [dict(d=96), dict(rot=0), dict(rot=24), dict(rot=144), dict(t=-1), dict(hq=0), dict(hkv=0), dict(max_pos=0),
        dict(dt=2), dict(q_ts=1000), dict(q_ts=1028), dict(k_ts=248), dict(v_ts=260), dict(q_out=None), dict(q=None),
        dict(k=None), dict(v=None), dict(cs=None), dict(pos=None), dict(kc=None), dict(vc=None), dict(slots=None),
        dict(bs=0), dict(fmt=4), dict(layout=2), dict(stride=16 * 2 * 256 - 16), dict(stride=16 * 2 * 256 + 8),
        dict(q=C.c_void_p(4104)), dict(kc=C.c_void_p(4104)), dict(kc=C.c_void_p(4097), fmt=2),
        dict(t=1 << 27)]


@pytest.mark.parametrize("call,cases", [(_prefix, PREFIX), (_cross, CROSS), (_rope, ROPE)])
def test_refused(call, cases):
    from vm_c_amd import capi
    lib = capi.load()
    for kw in cases:
        assert call(lib, **kw) == capi.VMC_EINVAL, kw


def test_nothing_to_do():
    from vm_c_amd import capi
    lib = capi.load()
    assert _prefix(lib, batch=0, out=None, q=None) == capi.VMC_OK
    assert _cross(lib, t=0, out=None) == capi.VMC_OK and _cross(lib, s=0, q=None) == capi.VMC_OK
    assert _rope(lib, t=0, q=None) == capi.VMC_OK


def _meta(*shape, dtype="float16"):
    import torch
    return torch.empty(shape, dtype=getattr(torch, dtype))


def test_binding_refuses():
    """Shapes, types and strides that the C side cannot see."""
    from vm_c_amd import capi
    i32, i64 = (lambda n: _meta(n, dtype="int32")), (lambda n: _meta(n, dtype="int64"))
    q, kv = _meta(4, 8, 128), _meta(100, 2, 128)
    bad = [dict(key=_meta(100, 2, 64)), dict(value=_meta(99, 2, 128)), dict(value=_meta(100, 2, 128, dtype="bfloat16")),
           dict(out=_meta(4, 8, 64)), dict(out=_meta(8, 4, 128).transpose(0, 1)), dict(query_starts=i32(2)),
           dict(key_starts=i32(3)), dict(key_lens=i64(2)), dict(query_starts=i64(3)),
           dict(key=_meta(100, 128, 2).transpose(1, 2))]
    for kw in bad:
        a = dict(out=_meta(4, 8, 128), query=q, key=kv, value=kv, query_starts=i32(3), key_starts=i32(2),
                 key_lens=i32(2), scale=0.1)
        a.update(kw)
        with pytest.raises(capi.VmcError):
            capi.cross_attention(**a)
    bad = [dict(group_starts=i32(2)), dict(group_starts=i64(3)), dict(seq_lens=i64(4)), dict(seq_lens=i32(3)),
           dict(out=_meta(4, 8, 64)), dict(query=_meta(8, 4, 128).transpose(0, 1)), dict(block_tables=_meta(4, 6)),
           dict(block_tables=_meta(3, 6, dtype="int32")), dict(shared_lens=i64(2))]
    for kw in bad:
        a = dict(out=_meta(4, 8, 128), query=q, key_cache=kv, value_cache=kv,
                 block_tables=_meta(4, 6, dtype="int32"), seq_lens=i32(4), group_starts=i32(3), shared_lens=i32(2),
                 num_kv_heads=2, scale=0.1)
        a.update(kw)
        with pytest.raises(capi.VmcError):
            capi.paged_attention_shared_prefix(**a)
    bad = [dict(key=_meta(3, 2, 128)), dict(value=_meta(4, 3, 128)), dict(key=_meta(4, 2, 128, dtype="bfloat16")),
           dict(cos_sin=_meta(50, 128)), dict(position_ids=i32(4)), dict(position_ids=i64(5)),
           dict(slot_mapping=i64(3)), dict(query_out=_meta(4, 8, 64)), dict(key_out=_meta(2, 4, 128).transpose(0, 1)),
           dict(query=_meta(8, 4, 128).transpose(0, 1))]
    for kw in bad:
        a = dict(query=q, key=_meta(4, 2, 128), value=_meta(4, 2, 128), cos_sin=_meta(50, 128, dtype="float32"),
                 position_ids=i64(4), key_cache=kv, value_cache=kv, slot_mapping=i64(4))
        a.update(kw)
        with pytest.raises(capi.VmcError):
            capi.rope_and_cache(**a)
