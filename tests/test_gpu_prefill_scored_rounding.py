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
