"""Rotary positions against their definition in 64 bits, and their fused forms against the separate calls.

Tolerance.  Angle: 2^-33 turns from the fixed point (4.6e-10 rad per half step), half a step of an fp32
value of at most an eighth of a turn (pi/4 * 2^-24 = 4.7e-8).  sincospi: at most 2 ulp of a value up to 1
(2^-22 at the most).  Amplitude, product and sum: three roundings of 2^-24.  Together below
amplitude * (|x0| + |x1|) * 2^-21, plus half a step of the output type.
"""
import math

import numpy as np
import pytest

from paged_fixture import load_b200

pytestmark = pytest.mark.gpu

SCALINGS = {
    "none": {}, "linear": dict(factor=4.0), "base": dict(factor=8.0),
    "ramp": dict(factor=16.0, orig_context=4096.0, low=1.0, high=32.0, amplitude=float(np.float32(0.1 * math.log(16.0) + 1.0))),
    "bands": dict(factor=8.0, orig_context=8192.0, low=1.0, high=4.0),
}


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


TWO_PI = 8 * np.arctan(np.longdouble(1))  # (64-bit mantissas: positions go up to 2^31)


def frequencies(scaling, r, theta, factor=1.0, orig_context=0.0, low=0.0, high=0.0, amplitude=1.0):
    i, theta = np.arange(r // 2, dtype=np.longdouble), np.longdouble(theta)
    if scaling == "base" and r > 2:
        theta = theta * np.longdouble(factor) ** (np.longdouble(r) / (r - 2))
    f = theta ** (-2 * i / r)
    if scaling == "linear":
        f = f / factor
    if scaling == "ramp":
        x = lambda turns: r * math.log(orig_context / (2 * math.pi * turns)) / (2 * math.log(float(theta)))
        a, z = max(math.floor(x(high)), 0), min(math.ceil(x(low)), r - 1)
        m = np.clip((i - a) / ((z - a) or 0.001), 0, 1)
        f = f / factor * m + f * (1 - m)
    if scaling == "bands":
        m = np.clip((orig_context * f / TWO_PI - low) / (high - low), 0, 1)
        f = f / factor * (1 - m) + f * m
    return f


def rotate(x, pos, layout, r, theta, scaling, **kw):
    """x [rows, heads, hd] float64; returns the rotated rows and the bound's |x0| + |x1| per element."""
    amp = kw.get("amplitude", 1.0)
    ang = np.outer(pos.astype(np.longdouble), frequencies(scaling, r, theta, **kw))[:, None]
    ang = (ang - np.rint(ang / TWO_PI) * TWO_PI).astype(np.float64)
    c, s = np.cos(ang), np.sin(ang)
    i = np.arange(r // 2)
    a, z = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y, size = x.copy(), np.zeros_like(x)
    y[..., a] = amp * (x[..., a] * c - x[..., z] * s)
    y[..., z] = amp * (x[..., a] * s + x[..., z] * c)
    size[..., a] = size[..., z] = amp * (np.abs(x[..., a]) + np.abs(x[..., z]))
    return y, size


def half_step(torch, t):
    return torch.finfo(t.dtype).eps / 2


def check(torch, got, want, size):
    """got: device tensor of `want`'s shape."""
    g = got.double().cpu().numpy().reshape(want.shape)
    bound = size * 2.0 ** -21 + np.abs(want) * half_step(torch, got) * 1.001 + 1e-30
    worst = (np.abs(g - want) / bound).max()
    assert worst <= 1.0, worst


def positions(torch, rng, rows, far):
    p = rng.integers(-far, far, rows)
    p[0] = far - 1
    if rows > 1:
        p[1] = 0
    return p, torch.tensor(p, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("scaling", list(SCALINGS))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,heads,kvh,hd,r,far", [
    (1, 10, 10, 128, 128, 1 << 31),    # one token, any position
    (64, 10, 10, 128, 64, 20000),
    (37, 4, 2, 64, 48, 1000000),
    (5, 3, 1, 80, 40, 300000),         # half layout: the halves are not whole chunks
    (9, 2, 2, 10, 6, 5000),            # rows that are not a multiple of 16 bytes
    (3, 1, 1, 2, 2, 100), (7, 1, 0, 256, 256, 65536), (4, 0, 3, 16, 2, 65536), (2500, 2, 1, 32, 32, 65536),
    (3, 2, 1, 512, 256, 65536), (2, 1, 2, 1024, 64, 65536), (2400, 3, 1, 264, 128, 4000),  # heads wider than a warp's 32 chunks
])
def test_rope_rows(b, scaling, layout, dtype, rows, heads, kvh, hd, r, far):
    import torch
    rng = np.random.default_rng(rows * 131 + hd + r)
    kw = SCALINGS[scaling]
    rope = b.Rope(layout=layout, rotary_dim=r, theta=10000.0, scaling=scaling, **kw)
    pos, d_pos = positions(torch, rng, rows, far)
    make = lambda n: torch.tensor(rng.standard_normal((rows, n * hd)), device="cuda").to(getattr(torch, dtype)) if n else None
    q, k = make(heads), make(kvh)
    q_out, k_out = (torch.full_like(t, float("nan")) if t is not None else None for t in (q, k))
    b.rope_rows(rope, q, k, q_out, k_out, d_pos, heads, kvh, hd)
    for x, out in ((q, q_out), (k, k_out)):
        if x is not None:
            want, size = rotate(x.double().cpu().numpy().reshape(rows, -1, hd), pos, layout, r, 10000.0, scaling, **kw)
            check(torch, out, want, size)
    # in place: the same bits
    for x, out in ((q, q_out), (k, k_out)):
        if x is not None:
            y = x.clone()
            if x is q:
                b.rope_rows(rope, y, None, y, None, d_pos, heads, 0, hd)
            else:
                b.rope_rows(rope, None, y, None, y, d_pos, 0, kvh, hd)
            assert torch.equal(y, out)


def test_rope_rows_strided_projection(b):
    """q, k, v inside one projection row, outputs inside wider rows, an odd (unaligned) one too."""
    import torch
    rng = np.random.default_rng(5)
    rows, heads, kvh, hd = 33, 4, 2, 64
    rope = b.Rope(layout="half", rotary_dim=64)
    pos, d_pos = positions(torch, rng, rows, 70000)
    for pad in (0, 8, 3):
        w = (heads + 2 * kvh) * hd + pad
        qkv = torch.tensor(rng.standard_normal((rows, w + pad)), device="cuda").float()
        q, k = qkv[:, pad:pad + heads * hd], qkv[:, pad + heads * hd:pad + (heads + kvh) * hd]
        before = qkv.clone()
        room = torch.full((rows, heads * hd + 24 + pad), 7.0, device="cuda")
        k_out = torch.full((rows, kvh * hd), float("nan"), device="cuda")
        b.rope_rows(rope, q, k, room[:, 16 + pad:16 + pad + heads * hd], k_out, d_pos, heads, kvh, hd)
        assert torch.equal(qkv, before)
        for x, out in ((q, room[:, 16 + pad:16 + pad + heads * hd]), (k, k_out)):
            want, size = rotate(x.double().cpu().numpy().reshape(rows, -1, hd), pos, "half", 64, 10000.0, "none")
            check(torch, out, want, size)
        assert (room[:, :16 + pad] == 7.0).all() and (room[:, 16 + pad + heads * hd:] == 7.0).all()


def paged(b, torch, rng, slots, blocks, kvh, hd, dtype, stride):
    ids = rng.permutation(blocks)[:slots * stride].reshape(slots, stride).astype(np.int32)
    table = torch.tensor(ids, device="cuda")
    layer = b.PagedLayer(blocks, kvh, hd, dtype, table)
    layer.k.fill_(3.0)
    layer.v.fill_(5.0)
    return layer, ids


@pytest.mark.parametrize("pool", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("layout,heads,kvh,hd,r", [("half", 4, 2, 64, 64), ("interleaved", 10, 10, 128, 64), ("half", 2, 1, 16, 10), ("half", 2, 2, 4, 4)])
@pytest.mark.parametrize("lens", [[1], [17, 0, 40], [900, 1, 1600]])
def test_rope_write_prefill(b, pool, dtype, layout, heads, kvh, hd, r, lens):
    """The fused write against rope_rows, and the pool's other tokens left as they were."""
    import torch
    if pool == "bf16" and hd < 8:
        pytest.skip("bf16 pools start at head_dim 8")
    rng = np.random.default_rng(sum(lens) + hd)
    rows = sum(lens)
    kd = b.BF16 if pool == "bf16" else b.F32
    stride = (max(lens) + 15) // 16
    layer, ids = paged(b, torch, rng, len(lens), len(lens) * stride + 3, kvh, hd, kd, stride)
    rope = b.Rope(layout=layout, rotary_dim=r, theta=1e6, scaling="linear", factor=2.0)
    pos, d_positions = positions(torch, rng, rows, 500000)
    slot = np.repeat(np.arange(len(lens)), lens)
    at = np.concatenate([np.arange(n) for n in lens])
    perm = rng.permutation(rows)
    ints = lambda x: torch.tensor(x[perm], dtype=torch.int32, device="cuda")
    tdt = getattr(torch, dtype)
    qkv = torch.tensor(rng.standard_normal((rows, (heads + 2 * kvh) * hd)), device="cuda").to(tdt)
    q, k, v = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kvh) * hd], qkv[:, (heads + kvh) * hd:]
    q_out = torch.full((rows, heads * hd), float("nan"), dtype=tdt, device="cuda")
    ws = b.Workspace(8)
    b.rope_write_prefill_paged(layer, rope, q, k, v, q_out, d_positions, ints(slot), ints(at), heads, ws)
    assert ws.status() == 0
    q_ref = torch.empty_like(q_out)
    k_ref = torch.empty((rows, kvh * hd), device="cuda")
    b.rope_rows(rope, q, None, q_ref, None, d_positions, heads, 0, hd)
    b.rope_rows(rope, None, k.float().contiguous(), None, k_ref, d_positions, 0, kvh, hd)  # fp32 out: not yet rounded
    assert torch.equal(q_out, q_ref)
    want_k, want_v = torch.full_like(layer.k, 3.0), torch.full_like(layer.v, 5.0)
    blk = torch.tensor(ids[slot[perm], at[perm] // 16].astype(np.int64), device="cuda")
    off = torch.tensor(at[perm] % 16, device="cuda")
    want_k[blk, :, off] = k_ref.to(layer.k.dtype).reshape(rows, kvh, hd)
    want_v[blk, :, off] = v.float().to(layer.v.dtype).reshape(rows, kvh, hd)
    assert torch.equal(layer.k, want_k) and torch.equal(layer.v, want_v)


@pytest.mark.parametrize("pool", ["f32", "bf16"])
@pytest.mark.parametrize("P,W", [(0, 16), (17, 20), (40, 1)])
def test_rope_append_equals_rope_then_append(b, pool, P, W):
    import torch
    rng = np.random.default_rng(P + W)
    slots, heads, kvh, hd = 5, 4, 2, 64
    kd = b.BF16 if pool == "bf16" else b.F32
    stride = (P + 15) // 16 + (W + 15) // 16
    one, ids = paged(b, torch, rng, slots, slots * stride, kvh, hd, kd, stride)
    two = b.PagedLayer(slots * stride, kvh, hd, kd, one.table, pools=(one.k.clone(), one.v.clone()))
    d_pre = torch.full((slots,), P, dtype=torch.int32, device="cuda")
    cur = [(d_pre.clone(), torch.zeros(slots, dtype=torch.int32, device="cuda")) for _ in range(2)]
    rope = b.Rope(layout="interleaved", rotary_dim=32)
    ws = b.Workspace(8)
    for t in range(2 * W + 3):
        batch = [3, 0, 4, 1] if t % 3 else [2, 4]
        d_slots = torch.tensor(batch, dtype=torch.int32, device="cuda")
        x = torch.tensor(rng.standard_normal((len(batch), (heads + 2 * kvh) * hd)), device="cuda").float()
        q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kvh) * hd], x[:, (heads + kvh) * hd:]
        pos = torch.full((len(batch),), P + t, dtype=torch.int32, device="cuda")
        q1, q2, k2 = (torch.empty((len(batch), n * hd), device="cuda") for n in (heads, heads, kvh))
        b.rope_append_decode_batch_paged(one, rope, q, k, v, q1, pos, *cur[0], d_pre, d_slots, W, heads, ws)
        b.rope_rows(rope, q, k, q2, k2, pos, heads, kvh, hd)
        b.append_decode_batch_paged(two, k2, v.contiguous(), *cur[1], d_pre, d_slots, len(batch), W, ws)
        assert torch.equal(q1, q2)
        assert torch.equal(one.k, two.k) and torch.equal(one.v, two.v)
        assert all(torch.equal(a, z) for a, z in zip(*cur))
    assert ws.status() == 0


def test_rope_append_same_slot_twice_and_bad_blocks(b):
    import torch
    slots, kvh, hd, W = 3, 1, 32, 16
    table = torch.tensor([[0], [99], [-1]], dtype=torch.int32, device="cuda")  # slot 1: beyond the pool, slot 2: retired
    layer = b.PagedLayer(3, kvh, hd, b.F32, table)
    rope, ws = b.Rope(rotary_dim=32), b.Workspace(4)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    d_len, d_ring, d_pre = ints(0, 0, 0), ints(0, 0, 0), ints(0, 0, 0)
    x = torch.arange(4 * hd, device="cuda").float().reshape(4, hd)
    out = torch.empty_like(x)
    run = lambda s: b.rope_append_decode_batch_paged(layer, rope, x[:len(s)], x[:len(s)], x[:len(s)], out[:len(s)], ints(*range(len(s))),
                                                     d_len, d_ring, d_pre, ints(*s), W, 1, ws)
    run([0, 0, 0])
    assert ws.status() == b.STATUS_BAD_SLOT
    assert d_len.tolist() == [1, 0, 0] and torch.equal(layer.v[0, 0, 0], x[0]) and not layer.v[0, 0, 1:].any()
    ref = torch.empty_like(x)
    b.rope_rows(rope, x, None, ref, None, ints(0, 1, 2, 3), 1, 0, hd)
    assert torch.equal(out[:3], ref[:3])
    run([1, 2])
    assert ws.status() == b.STATUS_BAD_BLOCK
    assert not layer.k[1:].any() and not layer.v[1:].any()
    b.rope_write_prefill_paged(layer, rope, x[:2], x[:2], x[:2], out[:2], ints(0, 1), ints(0, 0), ints(16, -1), 1, ws)
    assert ws.status() == b.STATUS_BAD_SLOT and torch.equal(out[:2], ref[:2])


def test_rope_in_a_captured_graph(b):
    import torch
    rope = b.Rope(layout="half", rotary_dim=128)
    x = torch.randn(64, 1280, device="cuda")
    pos = torch.arange(64, dtype=torch.int32, device="cuda")
    out, want = torch.zeros_like(x), torch.zeros_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            b.rope_rows(rope, x, None, out, None, pos, 10, 0, 128)
    for step in range(3):
        x.normal_()
        pos += 1000
        g.replay()
        b.rope_rows(rope, x, None, want, None, pos, 10, 0, 128)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_rope_wants_tensors_of_the_current_device(b):
    import torch
    x, pos = torch.zeros(2, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        b.rope_rows(b.Rope(rotary_dim=64), x, None, x, None, pos, 1, 0, 64)
