"""Attention with modified scores where values or ranges are extreme."""
import pytest

from paged_fixture import load_b200
from test_gpu_prefill_scored import MODES, Wave, slopes_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("cap,bias,q_dtype,out", MODES)
def test_prefill_infinite_query_of_either_sign(b, cap, bias, q_dtype, out, sign):
    """An infinity in a query makes its scores +inf or -inf, by the sign of the key's element; either way the row is NaN, unless it sees nothing."""
    import torch
    w = Wave(b, torch, [(140, 0, 140, 0), (0, 0, 3, 1), (20, 0, 4, 0)], 2, 2, seed=41)
    one = w.layer.k.nan_to_num(0)  # every key has the same sign in dim 7
    one[..., 7] = 1.0
    w.layer.k.copy_(torch.where(torch.isnan(w.layer.k), w.layer.k, one))
    tk = w.text[0]
    tk.copy_(torch.where(torch.isnan(tk), tk, torch.where(torch.arange(128, device="cuda") == 7, torch.ones_like(tk), tk)))
    q = w.q.clone()
    bad = [0, 1, 127, 128, 139, 140, 142, 143, 146]
    q[bad, 7] = sign * float("inf")  # head 0
    q = q.to(getattr(torch, q_dtype))
    hi = torch.cat([torch.arange(1, 141), torch.zeros(3), torch.zeros(4)]).to(torch.int32).cuda()  # the last request's rows see nothing
    pos = torch.arange(w.total, dtype=torch.int32, device="cuda")
    ws = b.Workspace(64)
    ws.set_out_dtype(b.BF16 if out == "bfloat16" else b.F32)
    got = torch.full((w.total, 256), 7.0, dtype=getattr(torch, out), device="cuda")
    score = b.Score(softcap=cap, slopes=slopes_of(torch, 2) if bias else None, d_q_pos=pos, d_hi=hi)
    b.prefill_attention_scored_tc(w.layer, *w.text, w.text_blocks, score, q, w.d_prefill, w.tiles, 9, 2, got, ws)
    assert ws.status() == 0
    hurt = torch.zeros(w.total, dtype=torch.bool, device="cuda")
    hurt[bad] = True
    hurt[143:] = False
    assert torch.isnan(got[hurt][:, :128]).all() and torch.isfinite(got[~hurt]).all() and torch.isfinite(got[:, 128:]).all()
    assert not got[143:].any()


@pytest.mark.parametrize("change", ["hi", "lo", "default", "prefix", "empty"])
def test_plan_that_no_longer_covers_the_ranges_is_reported(b, change):
    """A plan is reused with other ranges or prefix lengths than it was made for: reported where a row sees a key that no row of its tile saw then."""
    import torch
    w = Wave(b, torch, [(300, 0, 200, 0), (300, 0, 60, 1)], 2, 2, seed=5)
    full = lambda v: torch.full((w.total,), v, dtype=torch.int32, device="cuda")
    ws = b.Workspace(64)
    out = torch.empty(w.total, 256, device="cuda")
    plan = lambda score: b.prefill_plan_scored_tc(score, w.tiles, w.d_prefill, 16, ws)

    def status(score):
        b.prefill_attention_scored_tc(w.layer, *w.text, w.text_blocks, score, w.q, w.d_prefill, w.tiles, 16, 2, out, ws, reuse_plan=True)
        return ws.status()
    narrow, wide = {
        "hi": (b.Score(d_hi=full(100)), b.Score(d_hi=full(101))),
        "lo": (b.Score(d_lo=full(40), d_hi=full(290)), b.Score(d_lo=full(39), d_hi=full(290))),
        "default": (b.Score(d_hi=full(16)), b.Score()),
        "prefix": (b.Score(d_hi=full(400)),) * 2,
        "empty": (b.Score(d_hi=full(0)), b.Score(d_lo=full(299), d_hi=full(300))),
    }[change]
    if change == "prefix":
        w.d_prefill.fill_(100)
    plan(narrow)
    assert status(narrow) == 0
    if change == "prefix":
        w.d_prefill.fill_(300)
    assert status(wide) == b.STATUS_BAD_SLOT
    plan(wide)
    assert status(wide) == 0
    want = out.clone()
    if change == "prefix":
        return
    # the other way round the plan covers more than is seen, and the result is that of a plan of its own
    plan(narrow)
    assert status(narrow) == 0
    own = out.clone()
    plan(wide)
    assert status(narrow) == 0 and torch.equal(out, own) and not torch.equal(out, want)


@pytest.mark.parametrize("cap", [1e6, 1e20, 1e30])
@pytest.mark.parametrize("heads,kvh,hd,pool", [(2, 2, 128, "bf16"), (8, 2, 128, "bf16"), (3, 1, 32, "f32")])
def test_caps_far_above_the_scores_say_nothing(b, heads, kvh, hd, pool, cap):
    """Up to the largest cap: the result is the one without, within the bound of that (20 roundings of a score) plus the tanh's 2 ulp
    (4 roundings of the score, so 24 / 20 of it)."""
    import torch
    from score_fixture import Caches, attend, check_out
    c = Caches([(90, 20, 0)], kvh, hd, b.BF16 if pool == "bf16" else b.F32, 24, seed=7)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    q = torch.randn(1, heads * hd, device="cuda") * 2
    ws, out = b.Workspace(1), torch.empty(1, heads * hd, device="cuda")
    b.attention_scored_batch_paged(c.layer, b.Score(softcap=cap), q, c.d_len, c.d_ring, c.d_prefill, ints(0), 1, 24, heads, out, ws)
    assert ws.status() == 0
    want, _, tol, _ = attend(q[0].double().cpu().numpy(), c.k[0], c.v[0], 0.0, heads, kvh, hd)
    check_out(torch, out[0], want, 1.2 * tol)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("heads,hd,pool,prefix", [(1, 64, "bf16", 20), (2, 128, "bf16", 20), (4, 64, "bf16", 20), (3, 16, "f32", 20), (1, 64, "f32", 3000), (4, 128, "bf16", 3000)])
def test_decode_infinite_query_of_either_sign(b, heads, hd, pool, prefix, sign):
    """Scores that are all +inf or all -inf leave inf - inf in the softmax: NaN, as a whole item and joined from pieces."""
    import torch
    from score_fixture import Caches
    c = Caches([(prefix, 5, 0)], 1, hd, b.BF16 if pool == "bf16" else b.F32, 16, seed=2)
    k = c.layer.k
    k[..., 3] = torch.where(torch.isnan(k[..., 3]), k[..., 3], torch.ones_like(k[..., 3]))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    q = torch.randn(2, heads * hd, device="cuda")
    q[0, 3] = sign * float("inf")  # row 0, head 0
    ws, out = b.Workspace(2), torch.zeros(2, heads * hd, device="cuda")
    b.attention_scored_batch_paged(c.layer, b.Score(), q, c.d_len, c.d_ring, c.d_prefill, ints(0, 0), 2, 16, heads, out, ws)
    assert ws.status() == 0
    assert torch.isnan(out[0, :hd]).all() and torch.isfinite(out[0, hd:]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("heads,hd,pool,parts", [(1, 64, "bf16", False), (3, 128, "bf16", False), (4, 64, "f32", False), (2, 64, "bf16", False), (2, 128, "bf16", False),
                                                 (4, 128, "bf16", True), (8, 64, "bf16", True)])
def test_visible_infinities(b, heads, hd, pool, parts):
    """An infinite value that a row sees is infinite in its result, or NaN where the operands go in bf16 parts; one that it does not see leaves no trace."""
    import torch
    from score_fixture import Caches
    c = Caches([(40, 5, 0)], 1, hd, b.BF16 if pool == "bf16" else b.F32, 16, seed=6)
    c.layer.v[int(c.table_np[0, 1]), 0, 4, 9] = float("inf")  # token 20
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    q = torch.randn(2, heads * hd, device="cuda")
    ws, out = b.Workspace(2), torch.zeros(2, heads, hd, device="cuda")
    score = b.Score(d_lo=ints(0, 21))  # both in the same tile: row 1 sees from the next token on
    b.attention_scored_batch_paged(c.layer, score, q, c.d_len, c.d_ring, c.d_prefill, ints(0, 0), 2, 16, heads, out.view(2, -1), ws)
    assert ws.status() == 0
    seen = out[0, :, 9]
    assert (torch.isnan(seen) if parts else seen == float("inf")).all()
    out[0, :, 9] = 0
    assert torch.isfinite(out).all()


def test_plan_for_a_region_that_has_become_shorter_is_reported(b):
    """Blocks behind the shorter region may hold anything by now, and the plan has them multiplied by zero."""
    import torch
    w = Wave(b, torch, [(300, 0, 200, 0), (300, 0, 60, 1)], 2, 2, seed=5)
    ws, out = b.Workspace(64), torch.empty(w.total, 256, device="cuda")
    hi = torch.full((w.total,), 50, dtype=torch.int32, device="cuda")
    for score, lens, want in ((b.Score(), 299, b.STATUS_BAD_SLOT), (b.Score(), 100, b.STATUS_BAD_SLOT), (b.Score(d_hi=hi), 49, b.STATUS_BAD_SLOT),
                              (b.Score(d_hi=hi), 50, 0), (b.Score(d_hi=hi), 200, 0)):
        w.d_prefill.fill_(300)
        b.prefill_plan_scored_tc(score, w.tiles, w.d_prefill, 16, ws)
        w.d_prefill.fill_(lens)
        b.prefill_attention_scored_tc(w.layer, *w.text, w.text_blocks, score, w.q, w.d_prefill, w.tiles, 16, 2, out, ws, reuse_plan=True)
        assert ws.status() == want, (lens, want)
