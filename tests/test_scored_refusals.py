"""Caps and scales that fp32 does not hold are refused before anything else is looked at (no GPU here)."""
import ctypes as C
import os

import pytest

from paged_fixture import load_b200


@pytest.fixture(scope="module")
def b():
    m = load_b200()
    if not os.path.exists(m.LIB_PATH):
        m.build()
    return m


def calls(b, **score):
    """(status, message) of every call that takes the descriptor; none has a workspace, so none can run."""
    L, fake = b.lib(), 0x1000
    kv = C.byref(b.PagedKV(fake, fake, fake, 4, 8, 2, 128, b.BF16))
    sc = C.byref(b.ScoreDesc(**{**dict(scale=0.0, softcap=0.0, slopes=None, d_q_pos=None, d_key_pos=None, key_pos_stride=0, d_lo=None, d_hi=None), **score}))
    tiles = (C.c_int32 * 6)(0, 4, 0, 0, 0, 0)
    for rc in (lambda: L.uocr_b200_rswa_attention_scored_batch_paged(kv, sc, fake, 0, fake, fake, fake, fake, 4, 16, 4, fake, None, None, None),
               lambda: L.uocr_b200_rswa_attention_scored_ragged_paged(kv, sc, fake, 0, fake, fake, fake, 4, 4, fake, None, None),
               lambda: L.uocr_b200_rswa_prefill_text_scored_paged(kv, fake, fake, 4, sc, fake, 0, fake, fake, fake, fake, 4, 16, 4, fake, None, None),
               lambda: L.uocr_b200_rswa_prefill_attention_scored_tc(kv, None, None, 0, sc, fake, 0, fake, tiles, 1, 16, 4, fake, None, None),
               lambda: L.uocr_b200_rswa_prefill_plan_scored_tc(sc, tiles, 1, fake, 16, None, None)):
        yield rc(), L.uocr_b200_last_error().decode()


@pytest.mark.parametrize("score,about", [
    (dict(softcap=2.4e38), "softcap"), (dict(softcap=3.4e38), "softcap"), (dict(softcap=1.1e30), "softcap"), (dict(softcap=float("inf")), "softcap"),
    (dict(softcap=9e-7), "softcap"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
    (dict(scale=3e38), "scale"), (dict(scale=-3e38), "scale"), (dict(scale=1e35, softcap=1e-6), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
])
def test_what_fp32_does_not_hold(b, score, about):
    for rc, said in calls(b, **score):
        assert rc == 1 and about in said, said


@pytest.mark.parametrize("score", [dict(), dict(softcap=1e-6), dict(softcap=200.0, scale=1e37), dict(scale=-1e37), dict(scale=1e-38), dict(scale=1e31, softcap=1e-6)])
def test_what_it_holds(b, score):
    for rc, said in calls(b, **score):
        assert rc == 1 and "null pointer" in said, said  # (the workspace)
