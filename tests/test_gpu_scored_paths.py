"""Attention with modified scores on the paths the other tests do not take: every instantiation for grouped heads of a bf16 cache, with and
without attention weights, and rows cut into so many pieces that their partials are joined on four levels."""
import numpy as np
import pytest

import test_gpu_scored as base
from paged_fixture import load_b200
from score_fixture import Caches, attend, check_out

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


@pytest.mark.parametrize("option", ["plain", "cap", "bias", "range", "cap bias range scale", "bias range keypos"])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 128), (6, 3, 128), (8, 1, 128), (7, 1, 64), (20, 5, 64)])
def test_decode_of_grouped_heads(b, option, heads, kvh, hd):
    base.test_decode(b, option, heads, kvh, hd, "bf16")


@pytest.mark.parametrize("heads,kvh,hd,pool", [(16, 4, 128, "bf16"), (4, 2, 128, "bf16"), (8, 2, 64, "bf16"), (6, 3, 64, "bf16"), (4, 1, 128, "f32"), (6, 2, 32, "f32")])
@pytest.mark.parametrize("decay", [0.0, 0.5])
def test_mass_of_grouped_heads(b, heads, kvh, hd, pool, decay):
    base.test_mass(b, heads, kvh, hd, pool, decay)


@pytest.mark.parametrize("heads,kvh,hd,pool", [(1, 1, 64, "f32"), (1, 1, 128, "bf16"), (2, 1, 128, "bf16"), (4, 1, 64, "bf16"), (4, 1, 32, "f32")])
@pytest.mark.parametrize("prefix", [10000, 24000])
def test_rows_of_more_than_512_pieces(b, heads, kvh, hd, pool, prefix):
    """One row and one KV head: a piece is one to two tiles, 626 to 1502 partials of one item; and the weights of its tokens."""
    import torch
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    W, rng = 16, np.random.default_rng(prefix + hd)
    c = Caches([(prefix, 9, 0)], kvh, hd, b.BF16 if pool == "bf16" else b.F32, W, seed=hd)
    q = torch.tensor(rng.standard_normal((1, heads * hd)), device="cuda").float()
    ws, out = b.Workspace(1), torch.full((1, heads * hd), float("nan"), device="cuda")
    weights = torch.zeros(1, prefix, device="cuda")
    for again in range(2):  # the counters of the joins are back at zero after a launch
        mass = b.Mass(None, weights, 1, heads, decay=0.0)
        b.attention_scored_batch_paged(c.layer, b.Score(softcap=20.0), q, c.d_len, c.d_ring, c.d_prefill, ints(0), 1, W, heads, out, ws, mass=mass)
        assert ws.status() == 0
        want, w, tol, w_tol = attend(q[0].double().cpu().numpy(), c.k[0], c.v[0], np.zeros(prefix + 9), heads, kvh, hd, 0.0, 20.0)
        check_out(torch, out[0], want, tol, again)
        got, full = weights[0].double().cpu().numpy(), w.sum(0)[:prefix]
        assert (np.abs(got - full) <= w_tol.sum(0)[:prefix] + 2.0 ** -24 * (2 * heads + 4) * full).all()
        out.fill_(float("nan"))
