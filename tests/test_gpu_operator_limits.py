"""The cache operators at offsets that pass 32 bits, on two streams at a time, and beside rows that are not theirs."""
import numpy as np
import pytest

from paged_fixture import load_b200
from score_fixture import Caches, attend, check_out

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


def ints(torch, v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("pool", ["bf16", "f32"])
def test_blocks_beyond_32_bit_offsets(b, pool):
    """A pool of more than 2^31 elements whose last blocks are the ones in use: written with rotation, appended to, attended by every
    call, moved, and moved in place."""
    import torch
    rng = np.random.default_rng(4)
    heads, kvh, hd, W, P = 2, 1, 128, 16, 70
    dt, tdt = (b.BF16, torch.bfloat16) if pool == "bf16" else (b.F32, torch.float32)
    total = (1 << 20) + 64  # blocks of 2^11 elements: the last 64 begin at 2^31 elements
    pools = tuple(torch.empty(total, kvh, 16, hd, dtype=tdt, device="cuda") for _ in range(2))
    for x in pools:
        x[-64:] = 0
        x[:64] = float("nan")  # (what an offset cut to 32 bits would reach)
    nb = (P + 15) // 16
    table = ints(torch, [np.arange(total - 1, total - 2 - nb, -1)])
    layer = b.PagedLayer(total, kvh, hd, dt, table, pools=pools)
    rope, ws = b.Rope(rotary_dim=128), b.Workspace(P)
    pos, slots = ints(torch, np.arange(P)), ints(torch, [0] * P)
    make = lambda n, w: torch.tensor(rng.standard_normal((n, w)), device="cuda").float()
    q, k, v = make(P, heads * hd), make(P, kvh * hd), make(P, kvh * hd)
    q_out, k_turned = torch.empty_like(q), torch.empty_like(k)
    b.rope_write_prefill_paged(layer, rope, q, k, v, q_out, pos, slots, pos, heads, ws)
    b.rope_rows(rope, None, k, None, k_turned, pos, 0, kvh, hd)
    d_len, d_ring, d_prefill = ints(torch, [P]), ints(torch, [0]), ints(torch, [P])
    q1, k1, v1 = make(1, heads * hd), make(1, kvh * hd), make(1, kvh * hd)
    q1_out, k1_turned, here = torch.empty_like(q1), torch.empty_like(k1), ints(torch, [P])
    b.rope_append_decode_batch_paged(layer, rope, q1, k1, v1, q1_out, here, d_len, d_ring, d_prefill, slots[:1], W, heads, ws)
    b.rope_rows(rope, None, k1, None, k1_turned, here, 0, kvh, hd)
    rounded = lambda t: t.to(tdt).double().cpu().numpy().reshape(-1, kvh, hd)
    kk, vv = np.concatenate([rounded(k_turned), rounded(k1_turned)]), np.concatenate([rounded(v), rounded(v1)])

    def decode(kk, vv):
        out, n = torch.full((1, heads * hd), float("nan"), device="cuda"), len(kk) - 1
        mass = b.Mass(None, torch.zeros(1, P, device="cuda"), 1, heads)
        b.attention_scored_batch_paged(layer, b.Score(softcap=20.0), q1_out, d_len, d_ring, d_prefill, slots[:1], 1, W, heads, out, ws, mass=mass)
        want, w, tol, w_tol = attend(q1_out[0].double().cpu().numpy(), kk, vv, np.zeros(n + 1), heads, kvh, hd, 0.0, 20.0)
        check_out(torch, out[0], want, tol)
        got = mass.keep[1][0, :n].double().cpu().numpy()
        assert (np.abs(got - w.sum(0)[:n]) <= w_tol.sum(0)[:n] + 2.0 ** -20 * w.sum(0)[:n]).all()
    decode(kk, vv)
    out = torch.full((P, heads * hd), float("nan"), device="cuda")
    b.attention_scored_ragged_paged(layer, b.Score(), q_out, d_prefill, slots, pos, P, heads, out, ws)
    for r in (0, 16, P - 1):
        want, _, tol, _ = attend(q_out[r].double().cpu().numpy(), kk[:r + 1], vv[:r + 1], np.zeros(r + 1), heads, kvh, hd)
        check_out(torch, out[r], want, tol, r)
    if pool == "bf16":
        tc = torch.full_like(out, float("nan"))
        b.prefill_attention_scored_tc(layer, None, None, 0, b.Score(), q_out, d_prefill, b.make_prefill_tiles([(0, P, 0, 0, 0, 0)]), 16, heads, tc, ws)
        # the split of Q moves a score of up to 10 by 10 * 2^-16 at most, a weight by twice that, P by 2^-16; values are below 5
        assert (tc - out).abs().max().item() <= 5 * (2 * 10 * 2.0 ** -16 + 2.0 ** -16)
    # text rows from a text pool of that size: the same pools, block0 near the end
    text = torch.full((P, heads * hd), float("nan"), device="cuda")
    asc = total - 40
    for x, rows in zip(pools, (kk[:P], vv[:P])):
        x[asc:asc + nb] = torch.tensor(np.concatenate([rows, np.zeros((nb * 16 - P, kvh, hd))]).reshape(nb, 16, kvh, hd), device="cuda").transpose(1, 2).to(tdt)
    none = ints(torch, [0] * P)
    b.prefill_text_scored_paged(layer, *pools, total, b.Score(d_hi=none), q_out, d_prefill, slots, pos, ints(torch, [asc] * P), P, 1000, heads, text, ws)
    for r in (0, 16, P - 1):
        want, _, tol, _ = attend(q_out[r].double().cpu().numpy(), kk[:r + 1], vv[:r + 1], np.zeros(r + 1), heads, kvh, hd)
        check_out(torch, text[r], want, tol, r)
    # moved to new blocks up there, then in place
    mass = torch.rand(1, P, device="cuda")
    lens = d_len.reshape(1, 1)
    for keep, new in ((40, ints(torch, [[total - 50, total - 52, total - 51]])), (20, None)):
        d_keep, count = torch.empty(1, keep, dtype=torch.int32, device="cuda"), ints(torch, [0])
        b.evict_select(mass, d_prefill, slots[:1], 1, keep, 1, 1, d_keep, count, ws)
        kept = d_keep[0].cpu().numpy()
        b.evict_compact_paged_layers([layer], d_prefill, slots[:1], 1, d_keep, count, new, ws)
        b.evict_publish(table, slots[:1], 1, d_keep, count, lens, d_prefill, W, new, mass, None, ws)
        kk, vv = (np.concatenate([x[kept], x[-1:]]) for x in (kk, vv))
        decode(kk, vv)
    assert ws.status() == 0 and torch.isnan(pools[0][:64]).all() and torch.isnan(pools[1][:64]).all()


def test_two_streams_at_a_time(b):
    """Calls of two threads of work that share pools and tables, each with its workspace and stream, leave the bits of calls one after the other."""
    import torch
    c = Caches([(700, 24, 5), (90, 3, 0), (0, 7, 0), (333, 24, 0)], 2, 64, b.BF16, 24, seed=8)
    batch = ints(torch, [0, 1, 2, 3])
    streams, spaces = [torch.cuda.Stream() for _ in range(2)], [b.Workspace(4) for _ in range(2)]
    qs = [torch.randn(4, 8 * 64, device="cuda") for _ in range(2)]
    weights = [[torch.zeros(4, 704, device="cuda") for _ in range(2)] for _ in range(2)]
    masses = [[b.Mass(m, m, 4, 8) for m in pair] for pair in weights]
    score = b.Score(softcap=9.0)

    def step(i, out, mass, stream):
        b.attention_scored_batch_paged(c.layer, score, qs[i], c.d_len, c.d_ring, c.d_prefill, batch, 4, 24, 8, out, spaces[i], mass=mass, stream=stream)
    outs = [[torch.zeros(4, 512, device="cuda") for _ in range(2)] for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            step(i, outs[0][i], masses[0][i], streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        for _ in range(20):
            step(i, outs[1][i], masses[1][i], None)
    torch.cuda.synchronize()
    for i in range(2):
        assert spaces[i].status() == 0
        assert torch.equal(outs[0][i], outs[1][i]) and torch.equal(weights[0][i], weights[1][i])


@pytest.mark.parametrize("rows", [3, 40, 600])
@pytest.mark.parametrize("out_dtype", ["float32", "bfloat16"])
def test_rows_behind_the_last(b, rows, out_dtype):
    """What stands behind the rows of a call stays, also when some of the rows see nothing."""
    import torch
    heads, kvh, hd = 4, 2, 64
    c = Caches([(50, 8, 0), (0, 0, 0), (20, 0, 0)], kvh, hd, b.BF16, 24, seed=rows)
    slots = ints(torch, [i % 3 for i in range(rows)])
    pos = ints(torch, [i % 20 for i in range(rows)])
    q = torch.randn(rows, heads * hd, device="cuda")
    ws = b.Workspace(rows)
    ws.set_out_dtype(b.BF16 if out_dtype == "bfloat16" else b.F32)
    empty = ints(torch, [0 if i % 2 else 50 for i in range(rows)])
    text = [torch.zeros(8, kvh, 16, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    calls = (lambda o: b.attention_scored_batch_paged(c.layer, b.Score(d_hi=empty), q, c.d_len, c.d_ring, c.d_prefill, slots, rows, 24, heads, o, ws),
             lambda o: b.attention_scored_ragged_paged(c.layer, b.Score(d_hi=empty), q, c.d_prefill, slots, pos, rows, heads, o, ws),
             lambda o: b.prefill_text_scored_paged(c.layer, *text, 8, b.Score(d_hi=empty), q, c.d_prefill, slots, pos, torch.zeros_like(pos), rows, 24, heads, o, ws))
    for call in calls:
        out = torch.full((rows + 5, heads * hd), 77.0, dtype=getattr(torch, out_dtype), device="cuda")
        call(out)
        assert ws.status() == 0 and (out[rows:] == 77).all() and torch.isfinite(out[:rows]).all() and not (out[:rows] == 77).any()
