"""Tensor-core prefill with modified scores: what its roundings cost, checked apart from one another."""
import pytest

from paged_fixture import load_b200
from test_gpu_prefill_scored import Wave, slopes_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


@pytest.mark.parametrize("cap,bias", [(0.0, False), (0.0, True), (5.0, False), (5.0, True)])
@pytest.mark.parametrize("q_dtype", ["float32", "bfloat16"])
def test_bf16_results_are_rounded_once(b, q_dtype, cap, bias):
    """A bf16 result is the fp32 one rounded: no rounding of the probabilities to one bf16 in between.  Bound: that of fp32
    results (probabilities as bf16 pairs, 2^-16) and half a step of the result (bf16 keeps 8 bits of a value: 2^-8 of it at
    most); a cap adds 2^-19 of itself to every score, twice in the quotient, of values of at most the largest one."""
    import torch
    w = Wave(b, torch, [(273, 0, 273, 0), (30, 0, 40, 1), (1, 0, 1, 0)], 4, 2, seed=17)
    q_pos = torch.cat([torch.arange(pos0, pos0 + n, device="cuda") + (p if kind else 0) for p, pos0, n, kind in w.requests])
    slopes = slopes_of(torch, 4) if bias else None
    score = b.Score(softcap=cap, slopes=slopes, d_q_pos=q_pos.to(torch.int32) if bias else None)
    q = w.q.to(getattr(torch, q_dtype))
    ws = b.Workspace(64)
    ws.set_out_dtype(b.BF16)
    got = torch.empty(w.total, 4 * 128, dtype=torch.bfloat16, device="cuda")
    b.prefill_attention_scored_tc(w.layer, *w.text, w.text_blocks, score, q, w.d_prefill, w.tiles, 33, 4, got, ws)
    assert ws.status() == 0
    for s, (p, pos0, n, kind) in enumerate(w.requests):
        r = w.rows[s]
        i = pos0 + torch.arange(n, device="cuda")
        hi = i + 1 if kind == 0 else torch.full((n,), p, device="cuda")
        want, tol = w.want(s, q[r], torch.zeros(n, device="cuda"), hi, 33, q_pos[r], cap, 128 ** -0.5, slopes.double() if bias else None,
                           q_dtype == "float32", True)
        top = max(x.abs().max().item() for x in (w.v[s], *([w.tv[s]] if kind else [])))
        bound = tol + 2 * cap * 2.0 ** -19 * top + 2.0 ** -8 * 1.001 * want.abs() + 1e-30
        worst = ((got[r].double() - want).abs() / bound).max().item()
        assert worst <= 1, (s, worst)


@pytest.mark.parametrize("span", [4.0, 1.2, 0.6])
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_what_the_cap_costs(b, out, span):
    """The tanh alone: row r sees keys 4 r + 1 and 4 r + 2 (one of each half of the powers), whose scores it has exactly: one product of
    two bf16 each, up to `span` times the cap.  With values 1 and -1 the result is tanh((y0 - y1) / 2) of the capped scores y, so errors of
    y by e leave at most e.

    Roundings of y, as parts of the cap, tanh = 1 - 2 / (1 + p) with p = e^2x: p off by 2^-22 (ex2) or, for half of the keys of bf16
    results, by 2.7e-6 (polynomial) moves the tanh by half of that at most; the power's argument, two roundings, by 2^-24; 1 + p, the products
    of the denominators, the reciprocal (2^-23) and its products are seven roundings of 2^-24 of 2 / (1 + p), which is at most 2 and, where
    it is above 1, no longer meets the first error in full; the last sum 2^-24.  Together below 2^-20, with the polynomial 2^-19.
    fp32 rows whose scores stay below 5/8 of the cap: a polynomial right to 2^-22 of the score (1.1e-8 and six roundings).
    The two powers of the softmax and the bf16 pairs of the weights: 2^-15; bf16 results half a step, 2^-8 of the result."""
    import torch
    cap, rows = 256.0, 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(span * 10))
    w = Wave(b, torch, [(4 * rows, 0, rows, 0)], 1, 1, seed=3, poison=0.0)
    # scores: q has one element per key, the key one element; the second score is near the first, so that the result is not saturated
    r = torch.arange(rows, device="cuda")
    a0 = (torch.rand(rows, generator=gen, device="cuda") * 2 - 1) * span * cap / 8
    a1 = a0 + (torch.rand(rows, generator=gen, device="cuda") * 2 - 1) * 0.1 * (r % 2)  # every other row: equal scores, the result is the error
    q = torch.zeros(rows, 128, device="cuda")
    q[r, (2 * r) % 128], q[r, (2 * r + 1) % 128] = a0.bfloat16().float(), a1.bfloat16().float()
    q = q.bfloat16()
    k, v = torch.zeros(4 * rows, 128, device="cuda"), torch.zeros(4 * rows, 128, device="cuda")
    k[4 * r + 1, (2 * r) % 128] = k[4 * r + 2, (2 * r + 1) % 128] = 8.0
    v[4 * r + 1], v[4 * r + 2] = 1.0, -1.0
    blk = w.table[0, :(4 * rows) // 16].long()
    for pool, x in ((w.layer.k, k), (w.layer.v, v)):
        pool[blk] = x.bfloat16().reshape(-1, 1, 16, 128)
    ints = lambda t: t.to(torch.int32).contiguous()
    score = b.Score(scale=1.0, softcap=cap, d_lo=ints(4 * r + 1), d_hi=ints(4 * r + 3))
    ws = b.Workspace(64)
    ws.set_out_dtype(b.BF16 if out == "bfloat16" else b.F32)
    got = torch.empty(rows, 128, dtype=getattr(torch, out), device="cuda")
    b.prefill_attention_scored_tc(w.layer, None, None, 0, score, q, w.d_prefill, w.tiles, 8, 1, got, ws)
    assert ws.status() == 0
    s0, s1 = (q.double()[r, (2 * r + i) % 128] * 8 for i in (0, 1))
    y0, y1 = cap * torch.tanh(s0 / cap), cap * torch.tanh(s1 / cap)
    want = torch.tanh((y0 - y1) / 2)
    if out == "float32":
        each = cap * 2.0 ** -20
        bound = torch.where(torch.maximum(s0.abs(), s1.abs()) < 0.62 * cap, 2.0 ** -22 * torch.maximum(s0.abs(), s1.abs()), torch.full_like(s0, each))
    else:
        bound = torch.full_like(s0, cap * 2.0 ** -19)
    bound = bound + 2.0 ** -15 + (2.0 ** -8 if out == "bfloat16" else 2.0 ** -24) * want.abs()
    off = (got.double() - want[:, None]).abs().amax(1)
    assert (off <= bound).all(), (off / bound).max().item()
