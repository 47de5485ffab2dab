"""Arguments the cache operators refuse, as far as they are checked before the device is looked at (no GPU here)."""
import ctypes as C

import pytest

from paged_fixture import load_b200


@pytest.fixture(scope="module")
def b():
    import os
    m = load_b200()
    if not os.path.exists(m.LIB_PATH):
        m.build()
    return m


GOOD = dict(layout="half", rotary_dim=64, theta=10000.0)


@pytest.mark.parametrize("change", [
    dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=258), dict(rotary_dim=-2), dict(theta=0.0), dict(theta=-1.0), dict(theta=float("nan")),
    dict(theta=float("inf")), dict(amplitude=0.0), dict(amplitude=float("nan")), dict(scaling="linear", factor=0.0),
    dict(scaling="base", factor=float("inf")), dict(scaling="ramp", factor=4.0, orig_context=0.0, low=1.0, high=32.0),
    dict(scaling="ramp", factor=4.0, orig_context=4096.0, low=32.0, high=1.0), dict(scaling="ramp", factor=4.0, orig_context=4096.0, low=0.0, high=1.0),
    dict(scaling="ramp", factor=4.0, orig_context=4096.0, low=1.0, high=32.0, theta=1.0),
    dict(scaling="bands", factor=4.0, orig_context=4096.0, low=4.0, high=4.0),
])
def test_rope_create_refuses(b, change):
    with pytest.raises(b.Error):
        b.Rope(**{**GOOD, **change})


def test_rope_create_unknown_enums(b):
    h = C.c_void_p()
    for layout, scaling in ((2, 0), (-1, 0), (0, 5), (0, -1)):
        desc = b.RopeDesc(layout, 64, scaling, 10000.0, 2.0, 4096.0, 1.0, 4.0, 1.0)
        assert b.lib().uocr_b200_rope_create(C.byref(desc), C.byref(h)) != 0
    assert b.lib().uocr_b200_rope_create(None, C.byref(h)) != 0
    assert b.lib().uocr_b200_rope_create(C.byref(b.RopeDesc(0, 64, 0, 10000.0, 1.0, 0.0, 0.0, 0.0, 1.0)), None) != 0
    assert b.lib().uocr_b200_rope_destroy(None) == 0


def test_rope_calls_refuse(b):
    rope = b.Rope(**GOOD)
    L = b.lib()
    fake = 0x1000  # never dereferenced: every call below is refused first
    ok = dict(q=fake, k=fake, v=fake, q_out=fake, q_stride=128, k_stride=128, v_stride=128, q_out_stride=128, dtype=0, heads=1)
    rows = lambda **kw: C.byref(b.QkvRows(**{**ok, **kw}))
    call = lambda r, kv_heads=1, head_dim=128, k_out=fake, k_out_stride=128, pos=fake, total=4, h=None: L.uocr_b200_rswa_rope_rows(
        rope.h if h is None else h, r, k_out, k_out_stride, pos, total, kv_heads, head_dim, None)
    assert call(rows(), total=0) == 0
    assert call(rows(), pos=None) == 1
    assert call(None) == 1
    assert call(rows(), h=0) == 1
    assert call(rows(dtype=2)) == 2
    assert call(rows(heads=-1)) == 1
    assert call(rows(heads=0), kv_heads=0) == 1
    assert call(rows(heads=5000)) == 1
    assert call(rows(q=None)) == 1
    assert call(rows(q_out=None)) == 1
    assert call(rows(), k_out=None) == 1
    assert call(rows(), head_dim=32) == 1          # smaller than the rotated dims
    assert call(rows(), head_dim=2048) == 1
    assert call(rows(q_stride=127)) == 1
    assert call(rows(q_out_stride=64)) == 1
    assert call(rows(k_stride=0)) == 1
    assert call(rows(), k_out_stride=1) == 1
    assert call(rows(q_stride=256)) == 1           # in place with two strides
    kv = b.PagedKV(fake, fake, fake, 4, 8, 1, 128, b.BF16)
    write = lambda v=kv, r=None, slots=fake, pos=fake: L.uocr_b200_rswa_rope_write_prefill_paged(
        C.byref(v) if v else None, rope.h, r or rows(), fake, slots, pos, 4, None, None)
    assert write(v=None) == 1
    assert write(slots=None) == 1
    assert write(pos=None) == 1
    assert write(r=rows(v=None)) == 1
    assert write(r=rows(v_stride=3)) == 1
    assert write(v=b.PagedKV(fake, fake, fake, 4, 8, 1, 96, b.BF16)) == 2
    assert write(v=b.PagedKV(fake + 8, fake, fake, 4, 8, 1, 128, b.BF16)) == 1
    app = lambda window=8, ln=fake: L.uocr_b200_rswa_rope_append_decode_batch_paged(
        C.byref(kv), rope.h, rows(), fake, ln, fake, fake, fake, 4, window, None, None)
    assert app(window=0) == 1
    assert app(ln=None) == 1


def test_scored_calls_refuse(b):
    L, fake = b.lib(), 0x1000
    kv = b.PagedKV(fake, fake, fake, 4, 8, 2, 128, b.BF16)
    ok = dict(scale=0.0, softcap=0.0, slopes=None, d_q_pos=None, d_key_pos=None, key_pos_stride=0, d_lo=None, d_hi=None)
    sc = lambda **kw: C.byref(b.ScoreDesc(**{**ok, **kw}))
    inf, nan = float("inf"), float("nan")

    def decode(score=None, v=kv, q=fake, q_dtype=0, ln=fake, ring=fake, pre=fake, slots=fake, batch=4, window=16, heads=4, out=fake, mass=None, ws=None):
        return L.uocr_b200_rswa_attention_scored_batch_paged(C.byref(v) if v else None, sc() if score is None else score, q, q_dtype, ln, ring, pre, slots,
                                                             batch, window, heads, out, mass, ws, None)
    assert decode(batch=0) == 0
    assert decode() == 1 and b"null" in L.uocr_b200_last_error()  # no workspace
    assert decode(ln=None) == 1 and decode(ring=None) == 1 and decode(window=0) == 1 and decode(v=None) == 1
    assert decode(v=b.PagedKV(fake, fake, fake, 4, 8, 2, 96, b.BF16)) == 2
    assert L.uocr_b200_rswa_attention_scored_ragged_paged(C.byref(kv), sc(), fake, 0, fake, fake, None, 4, 4, fake, None, None) == 1
    text = lambda kt=fake, blocks=4, window=4, b0=fake: L.uocr_b200_rswa_prefill_text_scored_paged(
        C.byref(kv), kt, fake, blocks, sc(), fake, 0, fake, fake, fake, b0, 4, window, 4, fake, None, None)
    assert text(kt=None) == 1 and text(kt=fake + 8) == 1 and text(blocks=0) == 1 and text(window=0) == 1 and text(b0=None) == 1
    assert L.uocr_b200_rswa_mass_scratch_bytes(0, 4, 4) == 0
    assert L.uocr_b200_rswa_mass_scratch_bytes(3, 2, 5) == 128 + 48
    assert L.uocr_b200_rswa_mass_scratch_bytes(60000, 100, 100000) == 4 * 60000 * 100 * 100000 + 8 * 60000 * 100


def test_evict_calls_refuse(b):
    L, fake = b.lib(), 0x1000
    select = lambda mass=fake, stride=8, pre=fake, n=2, keep=4, sinks=0, recent=0, out=fake, ln=fake: L.uocr_b200_rswa_evict_select(
        mass, stride, pre, fake, n, keep, sinks, recent, out, ln, None, None)
    assert select(n=0) == 0
    for kw in (dict(mass=None), dict(stride=0), dict(pre=None), dict(keep=0), dict(keep=-1), dict(sinks=-1), dict(recent=-1), dict(out=None), dict(ln=None)):
        assert select(**kw) == 1, kw
    views = (b.PagedKV * 2)(b.PagedKV(fake, fake, fake, 4, 8, 2, 128, b.BF16), b.PagedKV(fake, fake, fake, 4, 8, 2, 64, b.BF16))
    compact = lambda layers=1, keep=fake, stride=4, new=fake, new_stride=1, n=2: L.uocr_b200_rswa_evict_compact_paged_layers(
        views, layers, fake, fake, n, keep, stride, fake, new, new_stride, None, None)
    assert compact(n=0) == 0
    assert compact(layers=2) == 1 and compact(layers=0) == 1 and compact(layers=33) == 1  # two geometries; layer counts
    assert compact(keep=None) == 1 and compact(stride=0) == 1 and compact(new_stride=0) == 1 and compact(n=70000) == 2
    publish = lambda table=fake, keep=fake, ln=fake, window=4, layers=1, mass=None, ms=0, kp=None, ks=0, new=None, ns=0: L.uocr_b200_rswa_evict_publish(
        table, 4, fake, 2, keep, 4, fake, new, ns, ln, 8, layers, fake, window, mass, ms, kp, ks, None, None)
    for kw in (dict(table=None), dict(keep=None), dict(ln=None), dict(window=0), dict(layers=0), dict(mass=fake), dict(kp=fake), dict(new=fake)):
        assert publish(**kw) == 1, kw
