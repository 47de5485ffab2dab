"""Tensor-core prefill with modified scores against 64 bits.

Bound per output element, for a row with weights w over its visible keys:
  scores      fp32 queries are split into two bf16 (off by 2^-16 of each element), bf16 queries are exact; 128 products
              are summed in fp32 (at most 24 roundings of 2^-24 on the way); cap 2^-21 of itself; bias and differences
              one rounding each; ex2 2^-22
  weights     bf16 pairs 2^-16, or one bf16 2^-8 where the result is bf16
  sums        one rounding of 2^-23 per 8 keys
and half a step of the result's own type.  A relative error e of numerator and denominator counts twice.
"""
import numpy as np
import pytest

from paged_fixture import load_b200

pytestmark = pytest.mark.gpu
HD = 128


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


class Wave:
    """Requests (slot prefix, first row's position, row count, kind) on one bf16 layer; text requests have their own text tokens."""

    def __init__(self, b, torch, requests, heads, kvh, seed, poison=float("nan"), hidden=()):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.b, self.torch, self.requests, self.heads, self.kvh = b, torch, requests, heads, kvh
        rng = np.random.default_rng(seed)
        self.prefix = [r[0] for r in requests]
        nb = [(p + 15) // 16 for p in self.prefix]
        total = sum(nb) + 3
        ids = rng.permutation(total)
        table = np.full((len(requests), max(nb) + 1), -1, np.int32)
        pools = [torch.full((total, kvh, 16, HD), poison, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        self.k, self.v, at = [], [], 0
        for s, n in enumerate(nb):
            table[s, :n] = ids[at:at + n]
            at += n
            kv = [torch.randn(self.prefix[s], kvh, HD, generator=gen, device="cuda").bfloat16() for _ in range(2)]
            for x in kv:
                for slot, lo, hi in hidden:
                    if slot == s:
                        x[lo:hi] = poison
            t = torch.arange(self.prefix[s], device="cuda")
            blk = torch.tensor(table[s, :max(n, 1)].astype(np.int64), device="cuda")
            for x, pl in zip(kv, pools):
                if n:
                    pl[blk[t // 16], :, t % 16] = x
            self.k.append(kv[0].double())
            self.v.append(kv[1].double())
        self.table = torch.tensor(table, device="cuda")
        self.layer = b.PagedLayer(total, kvh, HD, b.BF16, self.table, pools=tuple(pools))
        self.d_prefill = torch.tensor(self.prefix, dtype=torch.int32, device="cuda")
        # text tokens of the text requests: all from 0 up to the last row
        self.tk, self.tv, self.block0, blocks = {}, {}, {}, 1
        for s, (_, pos0, n, kind) in enumerate(requests):
            if kind == 1:
                self.block0[s] = blocks
                blocks += (pos0 + n + 15) // 16
        self.text_blocks = blocks + 1
        self.text = [torch.full((blocks + 1, kvh, 16, HD), poison, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        self.rows, spec, row0 = [], [], 0
        for s, (_, pos0, n, kind) in enumerate(requests):
            if kind == 1:
                m = pos0 + n
                kv = [torch.randn(m, kvh, HD, generator=gen, device="cuda").bfloat16() for _ in range(2)]
                t = torch.arange(m, device="cuda")
                for x, pl in zip(kv, self.text):
                    pl[self.block0[s] + t // 16, :, t % 16] = x
                self.tk[s], self.tv[s] = kv[0].double(), kv[1].double()
            spec.append((row0, n, s, kind, pos0, self.block0.get(s, 0)))
            self.rows.append(slice(row0, row0 + n))
            row0 += n
        self.total = row0
        self.tiles = b.make_prefill_tiles(spec)
        self.q = torch.randn(row0, heads * HD, generator=gen, device="cuda") * 1.5
        self.gen = gen

    def want(self, s, q, lo, hi, W, q_pos, cap, scale, slopes, pair_q, pair_p):
        """Rows of request s in 64 bits and the bound of each element."""
        torch = self.torch
        p, pos0, n, kind = self.requests[s]
        k, v = self.k[s], self.v[s]
        t = torch.arange(p, device="cuda")
        vis = (t >= lo[:, None]) & (t < hi[:, None])
        dist = (q_pos[:, None] - t).abs()
        if kind == 1:
            i, j = pos0 + torch.arange(n, device="cuda")[:, None], torch.arange(pos0 + n, device="cuda")
            vis = torch.cat([vis, (j <= i) & (j > i - W)], 1)
            dist = torch.cat([dist, (i - j).abs()], 1)
            k, v = torch.cat([k, self.tk[s]]), torch.cat([v, self.tv[s]])
        g = self.heads // self.kvh
        outs, tols = [], []
        for h in range(self.heads):
            kk, vv, qq = k[:, h // g], v[:, h // g], q[:, h * HD:(h + 1) * HD].double()
            seen = vis.any(0)  # unseen keys may be NaN
            kk, vv = torch.where(seen[:, None], kk, torch.zeros_like(kk)), torch.where(seen[:, None], vv, torch.zeros_like(vv))
            x = qq @ kk.T * scale
            size = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~vis, 0).amax(1) if len(kk) else torch.zeros(n, device="cuda").double()
            if cap:
                x = cap * torch.tanh(x / cap)
            far = torch.zeros_like(x)
            if slopes is not None:
                far = slopes[h] * dist
                x = x - far
            x = x.masked_fill(~vis, -torch.inf)
            none = ~vis.any(1)
            m = x.amax(1, keepdim=True) if len(kk) else torch.zeros(n, 1, device="cuda").double()
            e = torch.exp(x - m.masked_fill(none[:, None], 0))
            w = e / e.sum(1, keepdim=True).clamp_min(1e-300)
            live = w > 2.0 ** -40  # what smaller weights contribute stays below every bound here
            big = lambda y: y.masked_fill(~(vis & live), 0).abs().amax(1) if len(kk) else torch.zeros(n, device="cuda").double()
            eps = size * ((2.0 ** -16 if pair_q else 0) + 26 * 2.0 ** -24) + cap * 2.0 ** -21 + 4 * 2.0 ** -24 * (big(far) + big(x.nan_to_num(neginf=0))) + 2.0 ** -21
            rel = 2 * eps + (2.0 ** -16 if pair_p else 2.0 ** -8) + (vis.sum(1) / 8 + 16) * 2.0 ** -23
            outs.append(w @ vv)
            tols.append(rel[:, None] * (w @ vv.abs()))
        return torch.cat(outs, 1), torch.cat(tols, 1)

    def run(self, lo=None, hi=None, W=1024, cap=0.0, scale=0.0, slopes=None, q_pos=None, q_dtype="float32", out="float32", reuse=False):
        torch, b = self.torch, self.b
        ints = lambda x: x.to(torch.int32).contiguous() if x is not None else None
        score = b.Score(scale=scale, softcap=cap, slopes=slopes, d_q_pos=ints(q_pos), d_lo=ints(lo), d_hi=ints(hi))
        q = self.q.to(getattr(torch, q_dtype))
        ws = b.Workspace(max(len(self.tiles), 64))
        ws.set_out_dtype(b.BF16 if out == "bfloat16" else b.F32)
        got = torch.full((self.total + 3, self.heads * HD), 99.0, dtype=getattr(torch, out), device="cuda")
        if reuse:
            b.prefill_plan_scored_tc(score, self.tiles, self.d_prefill, W, ws)
        b.prefill_attention_scored_tc(self.layer, *self.text, self.text_blocks, score, q, self.d_prefill, self.tiles, W, self.heads, got, ws,
                                      reuse_plan=reuse)
        assert ws.status() == 0
        assert (got[self.total:] == 99).all()  # rows behind the last
        for s, (p, pos0, n, kind) in enumerate(self.requests):
            r = self.rows[s]
            i = pos0 + torch.arange(n, device="cuda")
            row_lo = (lo[r] if lo is not None else torch.zeros(n, device="cuda")).clamp_min(0)
            row_hi = (hi[r] if hi is not None else (i + 1 if kind == 0 else torch.full((n,), p, device="cuda"))).clamp_max(p)
            pos = q_pos[r] if q_pos is not None else i
            want, tol = self.want(s, q[r], row_lo, row_hi, W, pos, cap, scale or HD ** -0.5, slopes.double() if slopes is not None else None,
                                  q_dtype == "float32", out == "float32")
            half = torch.finfo(got.dtype).eps / 2
            bound = tol + half * 1.001 * want.abs() + 1e-30
            assert torch.isfinite(got[r]).all(), s
            assert ((got[r].double() - want).abs() <= bound).all(), (s, ((got[r].double() - want).abs() / bound).max().item())
        return got


def slopes_of(torch, heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")


MODES = [(c, s, q, o) for c in (0.0, 12.0) for s in (False, True) for q in ("float32", "bfloat16") for o in ("float32", "bfloat16")]


@pytest.mark.parametrize("cap,bias,q_dtype,out", MODES)
def test_vision_causal_and_text(b, cap, bias, q_dtype, out):
    """Causal vision rows and text rows of odd lengths in one launch; NaN in every row of the pools that holds no token."""
    import torch
    w = Wave(b, torch, [(273, 0, 273, 0), (130, 0, 300, 1), (1, 0, 1, 0), (0, 0, 77, 1), (257, 200, 57, 0), (40, 500, 33, 1)], 4, 2, seed=3)
    q_pos = torch.cat([torch.arange(pos0, pos0 + n, device="cuda") + (p if kind else 0) for p, pos0, n, kind in w.requests])
    w.run(W=150, cap=cap, slopes=slopes_of(torch, 4) if bias else None, q_pos=q_pos if bias else None, q_dtype=q_dtype, out=out)


@pytest.mark.parametrize("W", [1, 16, 100, 128, 129, 1000])
def test_text_windows(b, W):
    import torch
    w = Wave(b, torch, [(33, 0, 400, 1), (128, 300, 129, 1), (16, 0, 1, 1)], 2, 2, seed=W)
    q_pos = torch.cat([torch.arange(pos0, pos0 + n, device="cuda") + p for p, pos0, n, kind in w.requests])
    w.run(W=W, cap=20.0, slopes=slopes_of(torch, 2), q_pos=q_pos)


@pytest.mark.parametrize("edges", [[0, 100, 273, 274, 700], [0, 128, 256, 700], [0, 7, 15, 16, 17, 33, 700], [0, 350, 350, 700]])
@pytest.mark.parametrize("q_dtype,out", [("bfloat16", "bfloat16"), ("float32", "float32")])
def test_pages_that_see_themselves(b, edges, q_dtype, out):
    import torch
    w = Wave(b, torch, [(700, 0, 700, 0), (90, 0, 90, 0)], 2, 1, seed=sum(edges))
    lo, hi = torch.zeros(790, dtype=torch.int64, device="cuda"), torch.full((790,), 90, dtype=torch.int64, device="cuda")
    for a, z in zip(edges, edges[1:]):
        lo[a:z], hi[a:z] = a, z
    w.run(lo=lo, hi=hi, cap=30.0, q_dtype=q_dtype, out=out)
    w.run(lo=lo, hi=torch.minimum(hi, torch.cat([torch.arange(700, device="cuda"), torch.arange(90, device="cuda")]) + 1), slopes=slopes_of(torch, 2), reuse=True)


@pytest.mark.parametrize("seed", range(4))
def test_any_ranges(b, seed):
    """Ranges that differ from row to row, reach outside the region, or are empty; text rows that see part of the region or none of it."""
    import torch
    rng = np.random.default_rng(seed)
    req = [(300, 0, 300, 0), (513, 17, 140, 1), (45, 0, 3, 0), (200, 0, 130, 1)]
    w = Wave(b, torch, req, 2, 2, seed=seed + 50, poison=0.0)
    lo, hi = [], []
    for p, _, n, kind in req:
        a, z = rng.integers(-20, p + 20, n), rng.integers(-20, p + 20, n)
        if seed % 2:
            a[:], z[:] = p // 3 + rng.integers(0, 5), p // 2
        a[: n // 5], z[: n // 5] = 10, 10
        lo.append(a)
        hi.append(z)
    as_t = lambda x: torch.tensor(np.concatenate(x), device="cuda")
    w.run(lo=as_t(lo), hi=as_t(hi), W=60, cap=9.0, slopes=slopes_of(torch, 2), q_pos=torch.arange(w.total, device="cuda") * 3, scale=-0.07 if seed == 3 else 0.11)


def test_rows_that_see_nothing(b):
    import torch
    w = Wave(b, torch, [(200, 0, 200, 0), (0, 0, 5, 0)], 2, 2, seed=8)
    none = torch.zeros(205, dtype=torch.int64, device="cuda")
    got = w.run(lo=none, hi=none)
    assert not got[:205].any()


@pytest.mark.parametrize("lo,hi", [(37, 90), (128, 250), (130, 131), (16, 32)])
def test_nan_outside_the_span(b, lo, hi):
    """Tokens of the region before and behind what any row sees are NaN, in the very blocks that are read."""
    import torch
    w = Wave(b, torch, [(260, 0, 150, 0)], 2, 2, seed=lo, hidden=[(0, 0, lo), (0, hi, 260)])
    full = lambda v: torch.full((150,), v, device="cuda")
    w.run(lo=full(lo), hi=full(hi), cap=15.0, slopes=slopes_of(torch, 2), q_dtype="bfloat16", out="bfloat16")
    w.run(lo=full(lo), hi=full(hi))


@pytest.mark.parametrize("cap,bias,q_dtype,out", MODES)
def test_nan_in_a_query_stays_in_its_row(b, cap, bias, q_dtype, out):
    import torch
    w = Wave(b, torch, [(200, 0, 200, 0), (60, 0, 140, 1), (0, 0, 1, 0)], 2, 2, seed=31)
    q_pos = torch.cat([torch.arange(200, device="cuda"), 60 + torch.arange(140, device="cuda"), torch.zeros(1, device="cuda")]).to(torch.int32)
    score = b.Score(softcap=cap, slopes=slopes_of(torch, 2) if bias else None, d_q_pos=q_pos)
    ws = b.Workspace(64)
    ws.set_out_dtype(b.BF16 if out == "bfloat16" else b.F32)
    bad = [0, 5, 127, 128, 199, 200, 339, 340]  # the last one sees nothing
    q, hurt = w.q.to(getattr(torch, q_dtype)), w.q.clone()
    for i, r in enumerate(bad):
        hurt[r, 128 + i * 7] = float("nan") if i % 2 else float("inf")  # head 1 only
    res = []
    for x in (q, hurt.to(q.dtype)):
        o = torch.full((341, 256), 7.0, dtype=getattr(torch, out), device="cuda")
        b.prefill_attention_scored_tc(w.layer, *w.text, w.text_blocks, score, x, w.d_prefill, w.tiles, 100, 2, o, ws)
        res.append(o)
    assert ws.status() == 0
    good = torch.ones(341, dtype=torch.bool, device="cuda")
    good[bad[:-1]] = False
    assert torch.isnan(res[1][~good][:, 128:]).all() and not res[1][340].any()
    assert torch.equal(res[0][good], res[1][good]) and torch.equal(res[0][:, :128], res[1][:, :128])


def test_against_the_call_for_any_geometry(b):
    """Many items per CTA, plan reused by two calls, results next to the CUDA-core call's."""
    import torch
    req = [(700, 0, 700, 0)] * 5 + [(500, 0, 900, 1)] * 5
    w = Wave(b, torch, req, 10, 10, seed=21)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    q_pos = [t + (p if kind else 0) for p, _, n, kind in req for t in range(n)]
    score = b.Score(softcap=18.0, slopes=slopes_of(torch, 10), d_q_pos=ints(q_pos))
    ws, gen = b.Workspace(w.total), b.Workspace(w.total)
    b.prefill_plan_scored_tc(score, w.tiles, w.d_prefill, 300, ws)
    out = [torch.full((w.total, 1280), float("nan"), device="cuda") for _ in range(3)]
    for o in out[:2]:
        b.prefill_attention_scored_tc(w.layer, *w.text, w.text_blocks, score, w.q, w.d_prefill, w.tiles, 300, 10, o, ws, reuse_plan=True)
    assert ws.status() == 0 and torch.equal(out[0], out[1])
    cut = 3500
    slots, pos = [s for s, r in enumerate(req) for _ in range(r[2])], [t for r in req for t in range(r[2])]
    b.attention_scored_ragged_paged(w.layer, b.Score(softcap=18.0, slopes=slopes_of(torch, 10)), w.q[:cut], w.d_prefill, ints(slots[:cut]), ints(pos[:cut]), cut, 10,
                                    out[2][:cut], gen)
    b.prefill_text_scored_paged(w.layer, *w.text, w.text_blocks, b.Score(softcap=18.0, slopes=slopes_of(torch, 10), d_q_pos=ints(q_pos[cut:])), w.q[cut:], w.d_prefill,
                                ints(slots[cut:]), ints(pos[cut:]), ints([w.block0[s] for s in slots[cut:]]), w.total - cut, 300, 10, out[2][cut:], gen)
    assert gen.status() == 0
    rel = ((out[0] - out[2]).double().norm() / out[2].double().norm()).item()
    # both near the exact result: the split of Q moves a score of up to 10 by 10 * 2^-16 at most, a weight by as much
    assert rel <= 10 * 2.0 ** -16 + 2.0 ** -16


def test_plans_are_not_mixed(b):
    import torch
    w = Wave(b, torch, [(140, 0, 140, 0)], 2, 2, seed=4)
    ws = b.Workspace(64)
    out = torch.empty(140, 256, device="cuda")
    scored = lambda **kw: b.prefill_attention_scored_tc(w.layer, None, None, 0, b.Score(), w.q, w.d_prefill, w.tiles, 64, 2, out, ws, reuse_plan=True, **kw)
    plain = lambda: b.prefill_attention_tc(w.layer, None, None, 0, w.q, w.d_prefill, w.tiles, 64, 2, out, ws, reuse_plan=True)
    with pytest.raises(b.Error):
        scored()
    b.prefill_plan_tc(w.tiles, w.d_prefill, 64, ws)
    plain()
    with pytest.raises(b.Error):
        scored()
    b.prefill_plan_scored_tc(b.Score(), w.tiles, w.d_prefill, 64, ws)
    scored()
    with pytest.raises(b.Error):
        plain()
    assert ws.status() == 0


def test_refusals(b):
    import torch
    w = Wave(b, torch, [(20, 0, 20, 0), (20, 0, 4, 1)], 2, 2, seed=5)
    ws, out = b.Workspace(64), torch.empty(24, 256, device="cuda")
    pos = torch.zeros(24, dtype=torch.int32, device="cuda")

    def call(score, layer=w.layer, text=w.text, heads=2, window=8, q=w.q):
        b.prefill_attention_scored_tc(layer, *text, w.text_blocks, score, q, w.d_prefill, w.tiles, window, heads, out, ws)
    bad = [dict(score=b.Score(softcap=300.0)), dict(score=b.Score(softcap=1e-7)), dict(score=b.Score(softcap=-1.0)), dict(score=b.Score(softcap=float("nan"))), dict(score=b.Score(scale=float("inf"))),
           dict(score=b.Score(d_key_pos=pos.reshape(2, 12).contiguous())), dict(score=b.Score(slopes=slopes_of(torch, 2))),  # text rows need their positions
           dict(score=b.Score(), text=(None, None)), dict(score=b.Score(), heads=3), dict(score=b.Score(), window=0)]
    for kw in bad:
        with pytest.raises(b.Error):
            call(**kw)
    with pytest.raises(ValueError):
        call(b.Score(), q=w.q.half())
    f32 = b.PagedLayer(8, 2, HD, b.F32, w.table)
    with pytest.raises(b.Error):
        call(b.Score(), layer=f32)
    # the calls for any geometry, with a real workspace
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    small = b.Workspace(2)
    o = torch.empty(4, 256, device="cuda")
    for kw in (dict(score=b.Score(softcap=1e-9)), dict(score=b.Score(softcap=-2.0)), dict(score=b.Score(scale=float("nan"))), dict(score=b.Score(slopes=slopes_of(torch, 2))), dict(heads=3), dict(batch=3)):
        a = dict(score=b.Score(), heads=2, batch=1) | kw
        with pytest.raises(b.Error):
            b.attention_scored_batch_paged(w.layer, a["score"], w.q, ints(20, 20), ints(0, 0), w.d_prefill, ints(0, 0, 0), a["batch"], 16, a["heads"], o, small)
    m = torch.zeros(2, 32, device="cuda")
    for change in (dict(stride=0), dict(decay=-1.0), dict(decay=float("nan")), dict(scratch=None), dict(scratch_bytes=8), dict(mass_out=None)):
        mass = b.Mass(None, m, 1, 2)
        for k, v in change.items():
            setattr(mass.desc, k, v)
        with pytest.raises(b.Error):
            b.attention_scored_batch_paged(w.layer, b.Score(), w.q, ints(20, 20), ints(0, 0), w.d_prefill, ints(0), 1, 16, 2, o, small, mass=mass)
    assert ws.status() == 0 and small.status() == 0


def test_bad_blocks_are_reported(b):
    import torch
    w = Wave(b, torch, [(200, 0, 50, 0)], 1, 1, seed=6)
    ws, out = b.Workspace(64), torch.empty(50, 128, device="cuda")
    w.table[0, 1] = 10 ** 6
    b.prefill_attention_scored_tc(w.layer, None, None, 0, b.Score(), w.q, w.d_prefill, w.tiles, 8, 1, out, ws)
    assert ws.status() == b.STATUS_BAD_BLOCK
    few = torch.full((50,), 16, dtype=torch.int32, device="cuda")
    b.prefill_attention_scored_tc(w.layer, None, None, 0, b.Score(d_hi=few), w.q, w.d_prefill, w.tiles, 8, 1, out, ws)  # not looked at
    assert ws.status() == 0


def test_waits_that_run_out(b):
    import torch
    w = Wave(b, torch, [(300, 0, 300, 0), (50, 0, 200, 1)], 2, 2, seed=7)
    ws, out, want = b.Workspace(64), torch.empty(500, 256, device="cuda"), torch.empty(500, 256, device="cuda")
    call = lambda o: b.prefill_attention_scored_tc(w.layer, *w.text, w.text_blocks, b.Score(softcap=9.0), w.q, w.d_prefill, w.tiles, 64, 2, o, ws)
    call(want)
    ws.set_wait_limit(0)
    call(out)
    assert ws.status() & b.STATUS_WAIT_TIMEOUT
    ws.set_wait_limit(1 << 22)
    call(out)
    assert ws.status() == 0 and torch.equal(out, want)
