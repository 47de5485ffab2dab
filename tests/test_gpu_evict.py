"""Eviction from the fixed region: selection, compaction (new blocks and in place), publication, and a run of them."""
import math

import numpy as np
import pytest

from paged_fixture import load_b200
from score_fixture import attend, check_out

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


def ints(torch, v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def choose(mass, p, keep, sinks, recent):
    key = [math.inf if i < sinks or i >= p - recent else (-math.inf if math.isnan(mass[i]) else float(mass[i])) for i in range(p)]
    nan = [math.isnan(mass[i]) and key[i] == -math.inf for i in range(p)]
    return sorted(sorted(range(p), key=lambda i: (-key[i], nan[i], i))[:keep])


@pytest.mark.parametrize("kind", ["random", "ties", "constant", "zeros", "special"])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (16, 4, 8), (100, 0, 64), (333, 16, 0), (2048, 1, 1), (5, 7, 9), (7, 1 << 30, 0)])
def test_select(b, kind, keep, sinks, recent):
    import torch
    rng = np.random.default_rng(keep + sinks)
    lens = [0, 1, 31, 32, 33, 273, 1000, 2048, 5000]
    stride = 5003
    mass = rng.standard_normal((len(lens), stride)).astype(np.float32)
    if kind == "ties":
        mass = np.round(mass * 2) / 2
    if kind == "constant":
        mass[:] = 0.25
    if kind == "zeros":
        mass = np.where(rng.random(mass.shape) < 0.9, np.float32(0.0), mass)
        mass = np.where(rng.random(mass.shape) < 0.3, -mass, mass).astype(np.float32)  # -0 and 0 are the same weight
    if kind == "special":
        pick = rng.integers(0, 8, mass.shape)
        for v, x in ((0, math.nan), (1, math.inf), (2, -math.inf), (3, 1e-42), (4, -1e-42), (5, 3e38)):
            mass[pick == v] = x
    order = rng.permutation(len(lens))
    n = len(lens)
    d_keep, d_len = torch.full((n, keep), -7, dtype=torch.int32, device="cuda"), torch.full((n,), -7, dtype=torch.int32, device="cuda")
    ws = b.Workspace(1)
    b.evict_select(torch.tensor(mass, device="cuda"), ints(torch, lens), ints(torch, order), n, keep, sinks, recent, d_keep, d_len, ws)
    assert ws.status() == 0
    got = d_keep.cpu().numpy()
    for i, s in enumerate(order):
        want = choose(mass[s], lens[s], keep, sinks, recent)
        assert d_len[i].item() == len(want)
        assert got[i, :len(want)].tolist() == want, (i, s, lens[s])
        assert (got[i, len(want):] == -1).all()


def test_select_long_region(b):
    """Longer than what stays in shared memory; and a region longer than the mass row."""
    import torch
    rng = np.random.default_rng(1)
    p, keep = 120001, 40000
    mass = np.round(rng.exponential(size=(1, p)) * 1000).astype(np.float32)
    ws = b.Workspace(1)
    for stride in (p, 50000):
        m = torch.tensor(mass[:, :stride].copy(), device="cuda")
        d_keep, d_len = torch.empty((1, keep), dtype=torch.int32, device="cuda"), ints(torch, [0])
        b.evict_select(m, ints(torch, [p]), ints(torch, [0]), 1, keep, 10, 10, d_keep, d_len, ws)
        assert ws.status() == (0 if stride == p else b.STATUS_BAD_SLOT)
        assert d_keep[0].tolist() == choose(mass[0], min(p, stride), keep, 10, 10)


def build(b, torch, rng, lens, ring, W, layers, kvh, hd, dtype, extra):
    """Slots with their own prefixes and rings on `layers` pools of random rows; `extra` unused blocks."""
    nb = [(p + 15) // 16 for p in lens]
    rb = (W + 15) // 16
    total = sum(nb) + rb * len(lens) + extra
    ids = rng.permutation(total).astype(np.int32)
    table = np.full((len(lens), max(nb) + rb), -1, np.int32)
    at = 0
    for s, n in enumerate(nb):
        table[s, :n + rb] = ids[at:at + n + rb]
        at += n + rb
    d_table = torch.tensor(table, device="cuda")
    lay = [b.PagedLayer(total, kvh, hd, dtype, d_table) for _ in range(layers)]
    for x in lay:
        x.k.normal_()
        x.v.normal_()
    state = dict(d_len=torch.tensor([[p + r for p, r in zip(lens, ring)]] * layers, dtype=torch.int32, device="cuda"), d_prefill=ints(torch, lens),
                 d_ring=torch.zeros((layers, len(lens)), dtype=torch.int32, device="cuda"))
    return lay, d_table, ids[at:], state


def rows(pool, blocks, n):
    """First n tokens of a list of blocks: [n, kv_heads, hd]"""
    return pool[blocks.long()].transpose(1, 2).flatten(0, 1)[:n]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kvh,hd,dtype,layers", [(2, 64, "bf16", 3), (1, 256, "f32", 1), (10, 128, "bf16", 2), (3, 4, "f32", 2), (5, 8, "bf16", 1)])
@pytest.mark.parametrize("keep", [1, 17, 300])
def test_compact_and_publish(b, in_place, kvh, hd, dtype, layers, keep):
    import torch
    rng = np.random.default_rng(keep + hd)
    lens, ring, W = [40, 0, 257, 1, 640, 33], [5, 20, 20, 0, 7, 20], 20
    lay, table, free, st = build(b, torch, rng, lens, ring, W, layers, kvh, hd, b.BF16 if dtype == "bf16" else b.F32, extra=6 * 20)
    before = [(x.k.clone(), x.v.clone()) for x in lay]
    old_table = table.clone()
    stride = 700
    mass = torch.rand(len(lens), stride, device="cuda")
    key_pos = torch.cumsum(torch.randint(1, 4, (len(lens), stride), device="cuda"), 1).to(torch.int32)
    old_mass, old_pos = mass.clone(), key_pos.clone()
    slots = [4, 2, 1, 0, 2]  # slot 2 twice, slots 3 and 5 not at all
    n, ds = len(slots), ints(torch, slots)
    d_keep, d_len = torch.empty((n, keep), dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    ws = b.Workspace(1)
    b.evict_select(mass, st["d_prefill"], ds, n, keep, 2, 3, d_keep, d_len, ws)
    new = None if in_place else torch.tensor(free[:n * 20].reshape(n, 20).copy(), device="cuda")
    b.evict_compact_paged_layers(lay, st["d_prefill"], ds, n, d_keep, d_len, new, ws)
    b.evict_publish(table, ds, n, d_keep, d_len, st["d_len"], st["d_prefill"], W, new, mass, key_pos, ws)
    assert ws.status() == 0
    rb = (W + 15) // 16
    touched = set()
    for i, s in enumerate(slots):
        if s in slots[:i]:
            continue
        k = d_len[i].item()
        assert k == min(keep, lens[s]) and st["d_prefill"][s].item() == k
        assert st["d_len"][:, s].tolist() == [k + ring[s]] * layers
        nb, ob = (k + 15) // 16, (lens[s] + 15) // 16
        row = table[s].tolist()
        assert row[:nb] == (old_table[s, :nb] if in_place else new[i, :nb]).tolist()
        assert row[nb:nb + rb] == old_table[s, ob:ob + rb].tolist() and all(x == -1 for x in row[nb + rb:])
        kept = d_keep[i, :k].long()
        assert torch.equal(mass[s, :k], old_mass[s, kept]) and torch.equal(key_pos[s, :k], old_pos[s, kept])
        assert not mass[s, k:lens[s]].any() and not key_pos[s, k:lens[s]].any()
        assert torch.equal(mass[s, lens[s]:], old_mass[s, lens[s]:])
        touched |= set(row[:nb])
        for l, x in enumerate(lay):
            for pool, old in zip((x.k, x.v), before[l]):
                assert torch.equal(rows(pool, table[s, :nb], k), rows(old, old_table[s, :ob], lens[s])[kept])
                # the ring, and the rows behind the last kept token, stand as they were
                assert torch.equal(pool[table[s, nb:nb + rb].long()], old[old_table[s, ob:ob + rb].long()])
                if k % 16 and not in_place:
                    assert torch.equal(pool[row[nb - 1], :, k % 16:], old[row[nb - 1], :, k % 16:])
    for s in (3, 5):
        assert torch.equal(table[s], old_table[s]) and st["d_prefill"][s].item() == lens[s] and torch.equal(mass[s], old_mass[s])
    dup = set() if in_place else set(new[4].tolist())  # the second entry of slot 2 wrote its own new blocks, nobody reads them
    others = torch.tensor([x for x in range(lay[0].k.shape[0]) if x not in touched and x not in dup], device="cuda")
    for l, x in enumerate(lay):
        if not in_place:
            assert torch.equal(x.k[others], before[l][0][others]) and torch.equal(x.v[others], before[l][1][others])


def test_compact_reports_bad_input(b):
    import torch
    rng = np.random.default_rng(0)
    lay, table, free, st = build(b, torch, rng, [40], [0], 16, 1, 1, 32, b.F32, extra=4)
    before = lay[0].k.clone()
    ws, ds = b.Workspace(1), ints(torch, [0])
    call = lambda keep, count, new: b.evict_compact_paged_layers(lay, st["d_prefill"], ds, 1, ints(torch, [keep]), ints(torch, [count]), new, ws)
    call([-1, 40, 100, 5], 4, ints(torch, [[int(free[0])]]))
    assert ws.status() == b.STATUS_BAD_SLOT
    assert torch.equal(lay[0].k[int(free[0]), :, 3], before[table[0, 0].item(), :, 5])
    assert torch.equal(lay[0].k[int(free[0]), :, :3], before[int(free[0]), :, :3])
    call([1, 2], 2, ints(torch, [[99]]))
    assert ws.status() == b.STATUS_BAD_BLOCK
    call([1, 2], 2, ints(torch, [[-1]]))
    assert ws.status() == b.STATUS_BAD_BLOCK
    call(list(range(20)), 20, ints(torch, [[int(free[1])]]))  # the second block is missing
    assert ws.status() == b.STATUS_BAD_BLOCK
    table[0, 1] = 1000
    call([1, 20], 2, None)
    assert ws.status() == b.STATUS_BAD_BLOCK


@pytest.mark.parametrize("pool", ["bf16", "f32"])
def test_run_of_the_operators(b, pool):
    """A document is written with its rotation, decoded over its pages, evicted twice (new blocks, then in place) by the
    weights that decode left, and decoded on: at every step the cache answers as the tokens it is said to hold."""
    import torch
    rng = np.random.default_rng(12)
    heads, kvh, hd, W, P, layers = 4, 2, 64, 32, 150, 2
    dt = b.BF16 if pool == "bf16" else b.F32
    tdt = torch.bfloat16 if pool == "bf16" else torch.float32
    slots = 2
    lay, table, free, st = build(b, torch, rng, [P, P], [0, 0], W, layers, kvh, hd, dt, extra=40)
    stride = 176
    key_pos = torch.arange(stride, dtype=torch.int32, device="cuda").repeat(slots, 1).contiguous()
    mass = torch.zeros(slots, stride, device="cuda")
    want_mass, mass_tol = np.zeros((slots, P)), np.zeros((slots, P))
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    rope, ws = b.Rope(layout="interleaved", rotary_dim=32, scaling="ramp", factor=4.0, orig_context=128.0, low=1.0, high=8.0), b.Workspace(2 * P)
    # the logical content of every slot and layer: positions and K / V rows of the fixed region, then of the window
    fixed = [[None] * layers for _ in range(slots)]
    text = [[[] for _ in range(layers)] for _ in range(slots)]
    turned = torch.empty(2 * P, kvh * hd, device="cuda")
    pos2 = ints(torch, list(range(P)) * 2)
    for l in range(layers):
        x = torch.tensor(rng.standard_normal((2 * P, (heads + 2 * kvh) * hd)), device="cuda").float()
        q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kvh) * hd], x[:, (heads + kvh) * hd:]
        q_out = torch.empty(2 * P, heads * hd, device="cuda")
        b.rope_write_prefill_paged(lay[l], rope, q, k, v, q_out, pos2, ints(torch, [0] * P + [1] * P), pos2, heads, ws)
        b.rope_rows(rope, None, k, None, turned, pos2, 0, kvh, hd)
        for s in range(slots):
            rows_of = lambda t: t[s * P:(s + 1) * P].to(tdt).double().cpu().numpy().reshape(P, kvh, hd)
            fixed[s][l] = (np.arange(P), rows_of(turned), rows_of(v))
    step, here = 0, P
    new = torch.tensor(free[:8].reshape(2, 4).copy(), device="cuda")
    for phase in range(3):
        for _ in range(20):
            batch = [1, 0]
            ds = ints(torch, batch)
            pos = torch.full((2,), here, dtype=torch.int32, device="cuda")
            region = len(fixed[0][0][0])
            span = [(0, region), (region // 3, region)]  # what row 0 (slot 1) and row 1 (slot 0) see
            score = b.Score(softcap=25.0, slopes=slopes, d_q_pos=pos, d_key_pos=key_pos, d_lo=ints(torch, [span[0][0], span[1][0]]),
                            d_hi=ints(torch, [span[0][1], span[1][1]]))
            for l in range(layers):
                x = torch.tensor(rng.standard_normal((2, (heads + 2 * kvh) * hd)), device="cuda").float()
                q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kvh) * hd], x[:, (heads + kvh) * hd:]
                q_out, out, k_t = torch.empty(2, heads * hd, device="cuda"), torch.empty(2, heads * hd, device="cuda"), torch.empty(2, kvh * hd, device="cuda")
                b.rope_append_decode_batch_paged(lay[l], rope, q, k, v, q_out, pos, st["d_len"][l], st["d_ring"][l], st["d_prefill"], ds, W, heads, ws)
                b.rope_rows(rope, None, k, None, k_t, pos, 0, kvh, hd)
                b.attention_scored_batch_paged(lay[l], score, q_out, st["d_len"][l], st["d_ring"][l], st["d_prefill"], ds, 2, W, heads, out, ws,
                                               mass=b.Mass(mass, mass, 2, heads))
                for i, s in enumerate(batch):
                    text[s][l].append((here, k_t[i].to(tdt).double().cpu().numpy().reshape(kvh, hd), v[i].to(tdt).double().cpu().numpy().reshape(kvh, hd)))
                    text[s][l] = text[s][l][-W:]
                    lo, hi = span[i]
                    at, fk, fv = fixed[s][l]
                    kk = np.concatenate([fk[lo:hi], np.stack([t[1] for t in text[s][l]])])
                    vv = np.concatenate([fv[lo:hi], np.stack([t[2] for t in text[s][l]])])
                    dist = here - np.r_[at[lo:hi], [t[0] for t in text[s][l]]]
                    want, w, tol, wt = attend(q_out[i].double().cpu().numpy(), kk, vv, dist, heads, kvh, hd, 0.0, 25.0, slopes.double().cpu().numpy())
                    check_out(torch, out[i], want, tol, (phase, here, l, s))
                    want_mass[s, lo:hi] += w.sum(0)[:hi - lo]
                    mass_tol[s, lo:hi] += wt.sum(0)[:hi - lo] + 2.0 ** -24 * (2 * heads + 2) * want_mass[s, lo:hi]
            here += 1
        region = len(fixed[0][0][0])
        assert (np.abs(mass[:, :region].double().cpu().numpy() - want_mass[:, :region]) <= mass_tol[:, :region] + 1e-30).all()
        if phase == 2:
            break
        keep = 61 if phase == 0 else 17
        both = ints(torch, [0, 1])
        d_keep, d_n = torch.empty((2, keep), dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
        m_before = mass.cpu().numpy()
        b.evict_select(mass, st["d_prefill"], both, 2, keep, 1, 2, d_keep, d_n, ws)
        blocks = new if phase == 0 else None
        b.evict_compact_paged_layers(lay, st["d_prefill"], both, 2, d_keep, d_n, blocks, ws)
        b.evict_publish(table, both, 2, d_keep, d_n, st["d_len"], st["d_prefill"], W, blocks, mass, key_pos, ws)
        for s in range(slots):
            kept = choose(m_before[s], region, keep, 1, 2)
            assert d_keep[s].tolist() == kept
            assert key_pos[s, :keep].tolist() == fixed[s][0][0][kept].tolist()
            want_mass[s, :keep], mass_tol[s, :keep] = want_mass[s, kept], mass_tol[s, kept]
            for l in range(layers):
                fixed[s][l] = tuple(x[kept] for x in fixed[s][l])
    assert ws.status() == 0


def test_captured_eviction(b):
    """The three calls in one captured graph, replayed on new weights."""
    import torch
    rng = np.random.default_rng(3)
    W, keep, layers = 16, 40, 2
    lens = [100, 77]
    lay, table, free, st = build(b, torch, rng, lens, [4, 9], W, layers, 2, 32, b.F32, extra=8)
    arr, ds = b.layer_array(lay), ints(torch, [1, 0])
    new = torch.tensor(free[:6].reshape(2, 3).copy(), device="cuda")
    mass = torch.rand(2, 112, device="cuda")
    d_keep, d_n = torch.empty((2, keep), dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    ws = b.Workspace(1)
    start = [x.clone() for x in (table, st["d_len"], st["d_prefill"])]
    old = [(x.k.clone(), x.v.clone()) for x in lay]

    def step():
        b.evict_select(mass, st["d_prefill"], ds, 2, keep, 1, 1, d_keep, d_n, ws)
        b.evict_compact_paged_layers(arr, st["d_prefill"], ds, 2, d_keep, d_n, new, ws)
        b.evict_publish(table, ds, 2, d_keep, d_n, st["d_len"], st["d_prefill"], W, new, None, None, ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            step()
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        for x, y in zip((table, st["d_len"], st["d_prefill"]), start):
            x.copy_(y)
        mass.uniform_()
        g.replay()
        torch.cuda.synchronize()
        assert ws.status() == 0 and st["d_prefill"].tolist() == [40, 40] and st["d_len"][1].tolist() == [44, 49]
        for i, slot in enumerate((1, 0)):
            kept = torch.tensor(choose(mass[slot].cpu().numpy(), lens[slot], keep, 1, 1), device="cuda")
            assert torch.equal(d_keep[i].long(), kept)
            for x, (k, v) in zip(lay, old):
                assert torch.equal(rows(x.k, table[slot, :3], keep), rows(k, start[0][slot, :7], lens[slot])[kept])
                assert torch.equal(rows(x.v, table[slot, :3], keep), rows(v, start[0][slot, :7], lens[slot])[kept])
