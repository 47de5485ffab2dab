"""Attention with modified scores (decode, vision rows, text rows, accumulated weights) against 64 bits."""
import numpy as np
import pytest

from paged_fixture import load_b200
from score_fixture import BT, Caches, attend, check_out

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


SLOTS = [(40, 20, 0), (0, 7, 0), (17, 0, 0), (33, 24, 5), (1, 24, 0), (0, 0, 0), (100, 24, 23), (16, 1, 0)]  # window 24
GEOMETRY = [(2, 2, 128), (4, 2, 64), (8, 2, 32), (6, 2, 16), (3, 1, 256), (4, 1, 8), (16, 2, 128), (12, 1, 64), (2, 1, 4), (4, 1, 256)]


def options(name, rng, rows, spans, heads, p_max):
    """(kwargs for attend, kwargs for Score on the host, ranges per row)"""
    cap = 15.0 if "cap" in name else 0.0
    scale = 0.31 if "scale" in name else 0.0
    slopes = (2.0 ** -np.arange(1, heads + 1)).astype(np.float32).astype(np.float64) if "bias" in name else None
    ranges = None
    if "range" in name:
        ranges = []
        for r, p in enumerate(spans):
            lo = int(rng.integers(-3, p + 2))
            hi = int(rng.integers(lo - 2, p + 5))
            ranges.append((lo, hi) if r % 3 else (max(lo, 0), max(lo, 0)))
    return scale, cap, slopes, ranges


def ints(torch, v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("option", ["plain", "cap", "bias", "range", "cap bias range scale", "bias range keypos"])
@pytest.mark.parametrize("heads,kvh,hd", GEOMETRY)
@pytest.mark.parametrize("pool", ["bf16", "f32"])
def test_decode(b, option, heads, kvh, hd, pool):
    import torch
    if pool == "bf16" and hd < 8:
        pytest.skip("bf16 pools start at head_dim 8")
    rng = np.random.default_rng(heads * 1000 + hd)
    W = 24
    batch = [3, 0, 6, 5, 1, 2, 4, 7, 0, 6]  # slots in any order, two of them twice
    spans = [SLOTS[s][0] for s in batch]
    scale, cap, slopes, ranges = options(option, rng, len(batch), spans, heads, 100)
    seen = lambda i: (0, spans[i]) if ranges is None else (max(ranges[i][0], 0), min(ranges[i][1], spans[i]))
    hidden = {s: [t for t in range(SLOTS[s][0]) if not any(batch[i] == s and seen(i)[0] <= t < seen(i)[1] for i in range(len(batch)))]
              for s in set(batch)}
    c = Caches(SLOTS, kvh, hd, b.BF16 if pool == "bf16" else b.F32, W, seed=hd + heads, hidden=hidden)
    key_pos = np.cumsum(rng.integers(1, 5, (len(SLOTS), 100)), 1)
    q_pos = rng.integers(0, 600, len(batch))
    q_dtype = torch.bfloat16 if heads % 4 == 0 else torch.float32
    q = torch.tensor(rng.standard_normal((len(batch), heads * hd)) * 2, device="cuda").to(q_dtype)
    use_pos = "keypos" in option
    score = b.Score(scale=scale, softcap=cap, slopes=torch.tensor(slopes, dtype=torch.float32, device="cuda") if slopes is not None else None,
                    d_q_pos=ints(torch, q_pos) if slopes is not None else None, d_key_pos=ints(torch, key_pos) if use_pos else None,
                    d_lo=ints(torch, [x for x, _ in ranges]) if ranges else None, d_hi=ints(torch, [x for _, x in ranges]) if ranges else None)
    ws = b.Workspace(len(batch))
    qn = q.double().cpu().numpy()
    for out_dtype in (torch.float32, torch.bfloat16):
        ws.set_out_dtype(b.BF16 if out_dtype == torch.bfloat16 else b.F32)
        out = torch.full((len(batch), heads * hd), float("nan"), dtype=out_dtype, device="cuda")
        b.attention_scored_batch_paged(c.layer, score, q, c.d_len, c.d_ring, c.d_prefill, ints(torch, batch), len(batch), W, heads, out, ws)
        assert ws.status() == 0
        for i, s in enumerate(batch):
            lo, hi = seen(i)
            hi = max(lo, hi)
            p = spans[i]
            pick = np.r_[np.arange(lo, hi), np.arange(p, p + SLOTS[s][1])].astype(int)
            kp = key_pos[s] if use_pos else np.arange(100)
            dist = np.r_[q_pos[i] - kp[lo:hi], c.ring_age(s)]
            want, _, tol, _ = attend(qn[i], c.k[s][pick], c.v[s][pick], dist, heads, kvh, hd, scale, cap, slopes)
            check_out(torch, out[i], want, tol, (i, s))


def test_defaults_equal_the_plain_call(b):
    import torch
    c = Caches(SLOTS, 10, 128, b.BF16, 24, seed=3)
    batch = [0, 3, 6, 4]
    q = torch.randn(4, 1280, device="cuda")
    ws = b.Workspace(4)
    a, z = torch.empty_like(q), torch.empty_like(q)
    b.attention_scored_batch_paged(c.layer, b.Score(), q, c.d_len, c.d_ring, c.d_prefill, ints(torch, batch), 4, 24, 10, a, ws)
    b.attention_batch_paged(c.layer, q, c.d_len, c.d_prefill, ints(torch, batch), 4, 10, z, ws)
    # both are fp32 evaluations of the same formula: the bound the plain call is held to against the oracle
    assert (a - z).abs().max().item() <= 2e-5


@pytest.mark.parametrize("rows,prefix", [(1, 5000), (2, 777), (600, 30), (513, 16)])
def test_decode_sizes(b, rows, prefix):
    """One long cache cut over the whole GPU; batches planned in global memory."""
    import torch
    heads, kvh, hd, W = 4, 2, 64, 32
    rng = np.random.default_rng(rows)
    slots = [(prefix, 32, 3), (prefix // 2, 9, 0), (0, 0, 0)]
    c = Caches(slots, kvh, hd, b.BF16, W, seed=rows)
    batch = [i % 3 for i in range(rows)]
    q = torch.tensor(rng.standard_normal((rows, heads * hd)), device="cuda").float()
    slopes = np.array([0.5, 0.25, 0.0, 0.001])
    q_pos = np.full(rows, prefix + 50)
    score = b.Score(softcap=20.0, slopes=torch.tensor(slopes, dtype=torch.float32, device="cuda"), d_q_pos=ints(torch, q_pos))
    ws = b.Workspace(rows)
    out = torch.full((rows, heads * hd), float("nan"), device="cuda")
    b.attention_scored_batch_paged(c.layer, score, q, c.d_len, c.d_ring, c.d_prefill, ints(torch, batch), rows, W, heads, out, ws)
    assert ws.status() == 0
    for i in list(range(min(rows, 6))) + [rows - 1]:
        s = batch[i]
        p = slots[s][0]
        dist = np.r_[prefix + 50 - np.arange(p), c.ring_age(s)]
        sl = slopes.astype(np.float32).astype(np.float64)
        want, _, tol, _ = attend(q[i].double().cpu().numpy(), c.k[s], c.v[s], dist, heads, kvh, hd, 0.0, 20.0, sl)
        check_out(torch, out[i], want, tol, i)


@pytest.mark.parametrize("heads,kvh,hd,pool", [(10, 10, 128, "bf16"), (4, 2, 64, "f32"), (8, 1, 32, "bf16")])
@pytest.mark.parametrize("decay", [0.0, 1.0, 0.5])
def test_mass(b, heads, kvh, hd, pool, decay):
    import torch
    rng = np.random.default_rng(heads)
    batch = [3, 0, 6, 3, 5, 2, 6]  # slots 3 and 6 twice: their weights add up
    spans = [SLOTS[s][0] for s in batch]
    ranges = [(5, 20), (0, 40), (90, 100), (0, 33), (0, 0), (17, 3), (0, 50)]
    c = Caches(SLOTS, kvh, hd, b.BF16 if pool == "bf16" else b.F32, 24, seed=9)
    q = torch.tensor(rng.standard_normal((len(batch), heads * hd)), device="cuda").float()
    stride = 112
    start = rng.random((len(SLOTS), stride)).astype(np.float32)
    for same in (True, False):
        m_in = torch.tensor(start, device="cuda")
        if decay == 0.0:
            m_in.fill_(float("nan"))  # not read
        m_out = m_in if same else torch.full_like(m_in, -7.0)
        before = m_out.clone()
        mass = b.Mass(m_in, m_out, len(batch), heads, decay=decay)
        mass.scratch.fill_(255)  # NaN: nothing stale may be read
        score = b.Score(softcap=10.0, d_lo=ints(torch, [x for x, _ in ranges]), d_hi=ints(torch, [x for _, x in ranges]))
        ws = b.Workspace(len(batch))
        out = torch.empty_like(q)
        b.attention_scored_batch_paged(c.layer, score, q, c.d_len, c.d_ring, c.d_prefill, ints(torch, batch), len(batch), 24, heads, out, ws, mass=mass)
        assert ws.status() == 0
        want = np.zeros((len(SLOTS), stride))
        tol = np.zeros_like(want)
        for i, s in enumerate(batch):
            lo, hi = ranges[i][0], min(ranges[i][1], spans[i])
            hi = max(lo, hi) if hi > lo else lo
            pick = np.r_[np.arange(lo, hi), np.arange(spans[i], spans[i] + SLOTS[s][1])].astype(int)
            _, w, _, wt = attend(q[i].double().cpu().numpy(), c.k[s][pick], c.v[s][pick], np.zeros(len(pick)), heads, kvh, hd, 0.0, 10.0)
            want[s, lo:hi] += w.sum(0)[:hi - lo]
            tol[s, lo:hi] += wt.sum(0)[:hi - lo]
        got = m_out.double().cpu().numpy()
        for s in range(len(SLOTS)):
            p = SLOTS[s][0] if s in batch else 0
            full = want[s, :p] + (decay * start[s, :p] if decay else 0.0)
            bound = tol[s, :p] + 2.0 ** -24 * (2 * heads + 4) * np.abs(full) + 1e-30  # one rounding per term of the sum
            assert (np.abs(got[s, :p] - full) <= bound).all(), s
            left = before[s, p:].cpu().numpy()
            assert np.array_equal(m_out[s, p:].cpu().numpy(), left, equal_nan=True)
        again = m_out.clone()
        if not same:
            b.attention_scored_batch_paged(c.layer, score, q, c.d_len, c.d_ring, c.d_prefill, ints(torch, batch), len(batch), 24, heads, out, ws, mass=mass)
            assert np.array_equal(again.cpu().numpy(), m_out.cpu().numpy(), equal_nan=True)


def test_mass_stride_shorter_than_the_region(b):
    import torch
    c = Caches(SLOTS, 2, 64, b.F32, 24, seed=11)
    q = torch.randn(2, 128, device="cuda")
    ws, out = b.Workspace(2), torch.empty(2, 128, device="cuda")
    m = torch.zeros(len(SLOTS), 48, device="cuda")
    ref = torch.zeros(len(SLOTS), 112, device="cuda")
    for t in (m, ref):
        b.attention_scored_batch_paged(c.layer, b.Score(), q, c.d_len, c.d_ring, c.d_prefill, ints(torch, [6, 0]), 2, 24, 2, out, ws, mass=b.Mass(None, t, 2, 2))
        assert ws.status() == (b.STATUS_BAD_SLOT if t is m else 0)
    assert torch.equal(m, ref[:, :48])


@pytest.mark.parametrize("option", ["causal", "cap", "bias", "range", "cap bias range keypos"])
@pytest.mark.parametrize("heads,kvh,hd,pool", [(2, 2, 128, "bf16"), (4, 2, 64, "f32"), (8, 1, 16, "bf16")])
def test_ragged(b, option, heads, kvh, hd, pool):
    import torch
    rng = np.random.default_rng(hd)
    slots = [(37, 0, 0), (1, 0, 0), (50, 3, 0)]
    rows = [(0, t) for t in range(37)] + [(1, 0)] + [(2, t) for t in range(0, 50, 3)] + [(2, 60)]  # the last row lies behind the region
    rng.shuffle(rows)
    spans = [slots[s][0] for s, _ in rows]
    scale, cap, slopes, ranges = options(option, rng, len(rows), spans, heads, 50)
    c = Caches(slots, kvh, hd, b.BF16 if pool == "bf16" else b.F32, 16, seed=hd)
    key_pos = np.cumsum(rng.integers(1, 4, (3, 64)), 1)
    q = torch.tensor(rng.standard_normal((len(rows), heads * hd)), device="cuda").float()
    use_pos = "keypos" in option
    q_pos = np.array([key_pos[s][min(t, 63)] for s, t in rows]) if use_pos else np.array([t for _, t in rows])
    score = b.Score(softcap=cap, slopes=torch.tensor(slopes, dtype=torch.float32, device="cuda") if slopes is not None else None,
                    d_q_pos=ints(torch, q_pos) if use_pos else None, d_key_pos=ints(torch, key_pos) if use_pos else None,
                    d_lo=ints(torch, [x for x, _ in ranges]) if ranges else None, d_hi=ints(torch, [x for _, x in ranges]) if ranges else None)
    ws = b.Workspace(len(rows))
    out = torch.full((len(rows), heads * hd), float("nan"), device="cuda")
    b.attention_scored_ragged_paged(c.layer, score, q, c.d_prefill, ints(torch, [s for s, _ in rows]), ints(torch, [t for _, t in rows]), len(rows),
                                    heads, out, ws)
    assert ws.status() == 0
    for i, (s, t) in enumerate(rows):
        lo, hi = ranges[i] if ranges else (0, t + 1)
        lo, hi = max(lo, 0), min(hi, spans[i])
        hi = max(lo, hi)
        dist = q_pos[i] - (key_pos[s] if use_pos else np.arange(64))[lo:hi]
        want, _, tol, _ = attend(q[i].double().cpu().numpy(), c.k[s][lo:hi], c.v[s][lo:hi], dist, heads, kvh, hd, 0.0, cap, slopes)
        check_out(torch, out[i], want, tol, (i, s, t))


def text_pools(b, torch, rng, lens, kvh, hd, dtype):
    """A text pool with the requests' tokens one after the other, NaN where no token is; block0 per request, tokens in fp64."""
    tdt = torch.bfloat16 if dtype == b.BF16 else torch.float32
    blocks = sum((n + BT - 1) // BT for n in lens) + 1
    pools = [np.full((blocks, kvh, BT, hd), np.nan, np.float32) for _ in range(2)]
    toks, block0, at = [], [], 1
    for n in lens:
        block0.append(at)
        kv = [torch.tensor(rng.standard_normal((n, kvh, hd))).to(tdt).double().numpy() for _ in range(2)]
        for x, pl in zip(kv, pools):
            for t in range(n):
                pl[at + t // BT, :, t % BT] = x[t]
        toks.append(kv)
        at += (n + BT - 1) // BT
    return [torch.tensor(x, device="cuda").to(tdt) for x in pools], toks, block0, blocks


@pytest.mark.parametrize("option", ["plain", "cap", "bias", "range", "cap bias range keypos"])
@pytest.mark.parametrize("heads,kvh,hd,pool,W", [(2, 2, 128, "bf16", 20), (4, 2, 64, "f32", 1), (8, 1, 16, "bf16", 100)])
def test_text(b, option, heads, kvh, hd, pool, W):
    import torch
    rng = np.random.default_rng(hd + W)
    dt = b.BF16 if pool == "bf16" else b.F32
    slots = [(37, 0, 0), (0, 0, 0), (50, 0, 0)]
    lens = [33, 50, 1]
    c = Caches(slots, kvh, hd, dt, 16, seed=hd)
    (kt, vt), toks, block0, blocks = text_pools(b, torch, rng, lens, kvh, hd, dt)
    rows = [(s, t) for s in range(3) for t in range(lens[s])]
    rng.shuffle(rows)
    spans = [slots[s][0] for s, _ in rows]
    scale, cap, slopes, ranges = options(option, rng, len(rows), spans, heads, 50)
    key_pos = np.cumsum(rng.integers(1, 4, (3, 64)), 1)
    use_pos = "keypos" in option
    q = torch.tensor(rng.standard_normal((len(rows), heads * hd)), device="cuda").float()
    q_pos = np.array([(200 if use_pos else slots[s][0]) + t for s, t in rows])
    score = b.Score(softcap=cap, slopes=torch.tensor(slopes, dtype=torch.float32, device="cuda") if slopes is not None else None,
                    d_q_pos=ints(torch, q_pos), d_key_pos=ints(torch, key_pos) if use_pos else None,
                    d_lo=ints(torch, [x for x, _ in ranges]) if ranges else None, d_hi=ints(torch, [x for _, x in ranges]) if ranges else None)
    ws = b.Workspace(len(rows))
    out = torch.full((len(rows), heads * hd), float("nan"), device="cuda")
    b.prefill_text_scored_paged(c.layer, kt, vt, blocks, score, q, c.d_prefill, ints(torch, [s for s, _ in rows]), ints(torch, [t for _, t in rows]),
                                ints(torch, [block0[s] for s, _ in rows]), len(rows), W, heads, out, ws)
    assert ws.status() == 0
    for i, (s, t) in enumerate(rows):
        lo, hi = ranges[i] if ranges else (0, spans[i])
        lo, hi = max(lo, 0), min(hi, spans[i])
        hi = max(lo, hi)
        first = max(0, t - W + 1)
        k, v = (np.concatenate([x[s][lo:hi], toks[s][j][first:t + 1]]) for j, x in enumerate((c.k, c.v)))
        dist = np.r_[q_pos[i] - (key_pos[s] if use_pos else np.arange(64))[lo:hi], t - np.arange(first, t + 1)]
        want, _, tol, _ = attend(q[i].double().cpu().numpy(), k, v, dist, heads, kvh, hd, 0.0, cap, slopes)
        check_out(torch, out[i], want, tol, (i, s, t))


def test_visible_nan_and_infinite_scores(b):
    """What a row sees is not papered over: a visible NaN gives NaN, in its own row only."""
    import torch
    slots = [(20, 0, 0)]
    c = Caches(slots, 1, 64, b.BF16, 16, seed=1, hidden={0: [3]})
    q = torch.randn(2, 64, device="cuda")
    ws, out = b.Workspace(2), torch.empty(2, 64, device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        ws.set_out_dtype(b.BF16 if dt == torch.bfloat16 else b.F32)
        out = torch.empty(2, 64, dtype=dt, device="cuda")
        b.attention_scored_batch_paged(c.layer, b.Score(d_lo=ints(torch, [0, 4])), q, c.d_len, c.d_ring, c.d_prefill, ints(torch, [0, 0]), 2, 16, 1, out, ws)
        assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


def test_bad_blocks_are_reported(b):
    import torch
    c = Caches([(40, 0, 0)], 1, 64, b.F32, 16, seed=1)
    q, ws = torch.randn(1, 64, device="cuda"), b.Workspace(1)
    out = torch.empty(1, 64, device="cuda")
    call = lambda sc=b.Score(): b.attention_scored_batch_paged(c.layer, sc, q, c.d_len, c.d_ring, c.d_prefill, ints(torch, [0]), 1, 16, 1, out, ws)
    c.table[0, 1] = -1
    call()
    assert ws.status() == b.STATUS_BAD_BLOCK
    call(b.Score(d_hi=ints(torch, [16])))  # the bad block is not looked at
    assert ws.status() == 0
    c.table[0, 1] = 10 ** 6
    call()
    assert ws.status() == b.STATUS_BAD_BLOCK
    c.d_prefill[0] = c.d_len[0] = 16 * c.table.shape[1] + 1
    c.table[:] = 0
    call(b.Score(d_lo=ints(torch, [16 * c.table.shape[1]])))
    assert ws.status() & b.STATUS_BAD_SLOT


def test_waits_that_run_out(b):
    """With a poll limit of zero every wait gives up at once: status bit, no hang, and the workspace works again."""
    import torch
    c = Caches([(300, 16, 0)], 2, 128, b.BF16, 16, seed=1)
    q, ws = torch.randn(1, 256, device="cuda"), b.Workspace(1)
    out, want = torch.empty(1, 256, device="cuda"), torch.empty(1, 256, device="cuda")
    call = lambda o: b.attention_scored_batch_paged(c.layer, b.Score(softcap=5.0), q, c.d_len, c.d_ring, c.d_prefill, ints(torch, [0]), 1, 16, 2, o, ws)
    call(want)
    ws.set_wait_limit(0)
    call(out)
    assert ws.status() & b.STATUS_WAIT_TIMEOUT
    ws.set_wait_limit(1 << 22)
    call(out)
    assert ws.status() == 0 and torch.equal(out, want)


def test_captured_and_on_another_stream(b):
    import torch
    c = Caches(SLOTS, 4, 128, b.BF16, 24, seed=2)
    batch = ints(torch, [0, 3, 6])
    q = torch.randn(3, 512, device="cuda")
    ws, out, want = b.Workspace(3), torch.zeros(3, 512, device="cuda"), torch.zeros(3, 512, device="cuda")
    m, m2 = torch.zeros(len(SLOTS), 112, device="cuda"), torch.zeros(len(SLOTS), 112, device="cuda")
    mass, mass2 = b.Mass(m, m, 3, 4), b.Mass(m2, m2, 3, 4)
    score = b.Score(softcap=30.0)
    call = lambda o, ms: b.attention_scored_batch_paged(c.layer, score, q, c.d_len, c.d_ring, c.d_prefill, batch, 3, 24, 4, o, ws, mass=ms)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(out, mass)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(out, mass)
    torch.cuda.current_stream().wait_stream(s)
    call(want, mass2)
    for _ in range(3):
        q.normal_()
        g.replay()
        call(want, mass2)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(m, m2)


def test_text_blocks_outside_the_pool_are_reported(b):
    import torch
    c = Caches([(5, 0, 0)], 1, 64, b.F32, 16, seed=1)
    (kt, vt), _, block0, blocks = text_pools(b, torch, np.random.default_rng(0), [20], 1, 64, b.F32)
    q, ws = torch.randn(1, 64, device="cuda"), b.Workspace(1)
    out = torch.empty(1, 64, device="cuda")
    for at, bad in ((block0[0], False), (-1, True), (-(1 << 31), True), (blocks, True), ((1 << 31) - 1, True), (1 << 27, True)):
        b.prefill_text_scored_paged(c.layer, kt, vt, blocks, b.Score(), q, c.d_prefill, ints(torch, [0]), ints(torch, [19]), ints(torch, [at]), 1, 64, 1, out, ws)
        assert ws.status() == (b.STATUS_BAD_BLOCK if bad else 0), at
