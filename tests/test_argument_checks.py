"""Tensors that the calls of the cache operators would misread are refused in Python: the library gets bare addresses.

No GPU here: the tensors are on the CPU, the "current device" is theirs, and a stand-in for the library counts what reaches it."""
import os
from types import SimpleNamespace

import pytest
import torch

from paged_fixture import load_b200

KVH, HD, HEADS, N, SLOTS, STRIDE = 2, 64, 4, 6, 3, 40


@pytest.fixture()
def b(monkeypatch):
    m = load_b200()
    if not os.path.exists(m.LIB_PATH):
        m.build()
    rope, scratch = m.Rope(rotary_dim=32), m.lib().uocr_b200_rswa_mass_scratch_bytes
    reached = []

    class Library:
        uocr_b200_rswa_mass_scratch_bytes = staticmethod(scratch)

        def __getattr__(self, name):
            return lambda *a: reached.append((name, a)) or 0
    getattr(m, "_load_torch", lambda: None)()
    monkeypatch.setattr(m, "_current_device", lambda: -1, raising=False)
    monkeypatch.setattr(m, "_stream_of", lambda t, stream: 0, raising=False)
    monkeypatch.setattr(m, "lib", lambda: Library())
    return SimpleNamespace(m=m, rope=rope, reached=reached, ws=SimpleNamespace(h=1, out_dtype=m.F32, plan_rows=None), stream=SimpleNamespace(cuda_stream=0))


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def good(b):
    """Arguments of every call, by name."""
    m = b.m
    wide = torch.zeros(N, (HEADS + 2 * KVH) * HD)
    q, k, v = wide[:, :HEADS * HD], wide[:, HEADS * HD:(HEADS + KVH) * HD], wide[:, (HEADS + KVH) * HD:]
    layer = m.PagedLayer(5, KVH, HD, m.F32, ints(SLOTS, 4), device="cpu")
    score = m.Score(slopes=torch.zeros(HEADS), d_q_pos=ints(N), d_lo=ints(N), d_hi=ints(N))
    rows = dict(layer=layer, rope=b.rope, q=q, k=k, v=v, q_out=torch.zeros(N, HEADS * HD), d_positions=ints(N), d_slots=ints(N), heads=HEADS)
    att = dict(layer=layer, score=score, q=torch.zeros(N, HEADS * HD), d_prefill=ints(SLOTS), d_slots=ints(N), heads=HEADS, out=torch.zeros(N, HEADS * HD), ws=b.ws)
    text = dict(text_k=torch.zeros(2, KVH, 16, HD), text_v=torch.zeros(2, KVH, 16, HD), text_blocks=2)
    tiles = m.make_prefill_tiles([(0, N, 0, 0, 0, 0)])
    evict = dict(d_slots=ints(SLOTS), n=SLOTS, d_prefill=ints(SLOTS), d_keep=ints(SLOTS, 8), d_keep_len=ints(SLOTS))
    return {
        "rope_rows": dict(rope=b.rope, q=q, k=k, q_out=q, k_out=torch.zeros(N, KVH * HD), d_positions=ints(N), heads=HEADS, kv_heads=KVH, head_dim=HD),
        "rope_write_prefill_paged": dict(rows, d_pos=ints(N)),
        "rope_append_decode_batch_paged": dict(rows, d_len=ints(SLOTS), d_ring=ints(SLOTS), d_prefill=ints(SLOTS), window=16),
        "attention_scored_batch_paged": dict(att, d_len=ints(SLOTS), d_ring=ints(SLOTS), batch=N, window=16,
                                             mass=m.Mass(None, torch.zeros(SLOTS, STRIDE), N, HEADS)),
        "attention_scored_ragged_paged": dict(att, d_pos=ints(N), total=N),
        "prefill_text_scored_paged": dict(att, **text, d_pos=ints(N), d_block0=ints(N), total=N, window=16),
        "prefill_plan_scored_tc": dict(score=score, tiles=tiles, d_prefill=ints(SLOTS), window=16, ws=b.ws),
        "prefill_attention_scored_tc": dict({k: v for k, v in att.items() if k != "d_slots"}, **text, tiles=tiles, window=16),
        "evict_select": dict(evict, mass=torch.zeros(SLOTS, STRIDE), keep=8, sinks=1, recent=1),
        "evict_compact_paged_layers": dict(evict, layers=[layer], d_new_blocks=ints(SLOTS, 1)),
        "evict_publish": dict(evict, table=ints(SLOTS, 4), d_len=ints(2, SLOTS), window=16, d_new_blocks=ints(SLOTS, 1), mass=torch.zeros(SLOTS, STRIDE),
                              d_key_pos=ints(SLOTS, STRIDE)),
    }


CALLS = ["rope_rows", "rope_write_prefill_paged", "rope_append_decode_batch_paged", "attention_scored_batch_paged", "attention_scored_ragged_paged",
         "prefill_text_scored_paged", "prefill_plan_scored_tc", "prefill_attention_scored_tc", "evict_select", "evict_compact_paged_layers", "evict_publish"]


def call(b, name, **change):
    return getattr(b.m, name)(**{**good(b)[name], **change}, stream=b.stream)


@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_reach_the_library(b, name):
    call(b, name)
    assert [n for n, _ in b.reached] == ["uocr_b200_rswa_" + name]


@pytest.mark.parametrize("name", CALLS)
def test_integers_of_another_type(b, name):
    """int64 positions, slots, lengths, tables: read as int32 they are other numbers."""
    args = good(b)[name]
    seen = 0
    for key, t in args.items():
        if isinstance(t, torch.Tensor) and t.dtype == torch.int32:
            for bad in (t.long(), t.float()):
                with pytest.raises((b.m.Error, ValueError)):
                    call(b, name, **{key: bad})
                seen += 1
    assert seen and not b.reached


@pytest.mark.parametrize("name", CALLS)
def test_integers_that_are_too_few_or_strided(b, name):
    args = good(b)[name]
    for key, t in args.items():
        if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32) or (name == "evict_publish" and key == "d_len"):
            continue
        strided = torch.zeros(*t.shape, 2, dtype=torch.int32)[..., 0]
        with pytest.raises((b.m.Error, ValueError)):
            call(b, name, **{key: strided})
        if key not in ("d_len", "d_ring", "d_prefill", "table", "d_key_pos"):  # (how many slots there are is not known here)
            with pytest.raises((b.m.Error, ValueError)):
                call(b, name, **{key: t[:-1].contiguous()})
    assert not b.reached


@pytest.mark.parametrize("name", ["rope_rows", "rope_write_prefill_paged", "rope_append_decode_batch_paged"])
def test_rows_that_do_not_hold_the_heads(b, name):
    """A wide stride does not make a narrow matrix wide: the row's end would be read from, or written to, what lies behind it."""
    wide = torch.zeros(N, 4 * HEADS * HD)
    for key in ("q", "k", "v", "q_out", "k_out"):
        if good(b)[name].get(key) is None:
            continue
        width = (HEADS if key in ("q", "q_out") else KVH) * HD
        change = {key: wide[:, :width - 1]}
        if name == "rope_rows" and key == "q":
            change["q_out"] = torch.zeros(N, HEADS * HD)
        for bad in (wide[:, :width - 1], wide[:N - 1, :width], wide[:, :2 * width:2], wide.bfloat16()[:, :width] if key != "q" else wide.half()[:, :width], wide[0]):
            with pytest.raises((b.m.Error, ValueError)):
                call(b, name, **{**change, key: bad})
    assert not b.reached


@pytest.mark.parametrize("name", ["attention_scored_batch_paged", "attention_scored_ragged_paged", "prefill_text_scored_paged", "prefill_attention_scored_tc"])
def test_queries_and_results_of_attention(b, name):
    full = torch.zeros(N, HEADS * HD)
    bad = {"q": [full.half(), full[:-1], full[:, :-1].contiguous(), torch.zeros(N, 2 * HEADS * HD)[:, :HEADS * HD]],
           "out": [full.bfloat16(), full.half(), full.double(), full[:-1], torch.zeros(N, 2 * HEADS * HD)[:, :HEADS * HD]]}
    if "text_k" in good(b)[name]:
        pool = good(b)[name]["text_k"]
        bad["text_k"] = bad["text_v"] = [pool.bfloat16(), pool[:1], pool.transpose(1, 2)]
    for key, tensors in bad.items():
        for t in tensors:
            with pytest.raises((b.m.Error, ValueError)):
                call(b, name, **{key: t})
    b.ws.out_dtype = b.m.BF16  # a workspace that writes bf16
    with pytest.raises((b.m.Error, ValueError)):
        call(b, name)
    assert not b.reached
    call(b, name, out=full.bfloat16(), q=full.bfloat16())
    assert len(b.reached) == 1


@pytest.mark.parametrize("name", ["attention_scored_batch_paged", "attention_scored_ragged_paged", "prefill_text_scored_paged", "prefill_plan_scored_tc", "prefill_attention_scored_tc"])
def test_scores_for_fewer_rows_or_heads(b, name):
    few = ints(N - 1)
    scores = [dict(d_lo=few), dict(d_hi=few)]
    if name != "prefill_plan_scored_tc":
        scores += [dict(slopes=torch.zeros(HEADS), d_q_pos=few), dict(slopes=torch.zeros(HEADS - 1), d_q_pos=ints(N))]
    for kw in scores:
        with pytest.raises((b.m.Error, ValueError)):
            call(b, name, score=b.m.Score(**kw))
    assert not b.reached
    call(b, name, score=b.m.Score(d_q_pos=few))  # without a bias the positions are not read
    assert len(b.reached) == 1


def test_masses(b):
    for name in ("evict_select", "evict_publish"):
        for bad in (torch.zeros(SLOTS, STRIDE, dtype=torch.float64), torch.zeros(SLOTS, STRIDE).bfloat16(), torch.zeros(SLOTS, 2 * STRIDE)[:, :STRIDE], torch.zeros(STRIDE)):
            with pytest.raises((b.m.Error, ValueError)):
                call(b, name, mass=bad)
    with pytest.raises((b.m.Error, ValueError)):
        call(b, "evict_publish", d_len=ints(SLOTS, 2).T)
    with pytest.raises((b.m.Error, ValueError)):
        call(b, "evict_publish", d_len=ints(SLOTS))
    assert not b.reached


@pytest.mark.parametrize("name", CALLS)
def test_another_device(b, name, monkeypatch):
    monkeypatch.setattr(b.m, "_current_device", lambda: 0, raising=False)
    with pytest.raises((b.m.Error, ValueError)):
        call(b, name)
    assert not b.reached


def test_a_reused_plan_tells_the_rows(b):
    """With reuse_plan the rows that are read are those of the plan, not of the tiles given beside it."""
    args = good(b)["prefill_attention_scored_tc"]
    call(b, "prefill_plan_scored_tc", tiles=b.m.make_prefill_tiles([(0, 2 * N, 0, 0, 0, 0)]), score=b.m.Score())
    with pytest.raises((b.m.Error, ValueError)):
        call(b, "prefill_attention_scored_tc", reuse_plan=True)
    call(b, "prefill_plan_scored_tc")
    call(b, "prefill_attention_scored_tc", reuse_plan=True)
    assert [n for n, _ in b.reached][-1] == "uocr_b200_rswa_prefill_attention_scored_tc" and args["tiles"].shape == (1, 6)
    with pytest.raises((b.m.Error, ValueError)):
        call(b, "prefill_plan_scored_tc", tiles=b.m.make_prefill_tiles([(0, N, 0, 0, 0, 0)])[:, :5])


def test_one_row_in_place_from_two_views(b):
    """The stride of a single row says nothing: views of one row with different strides are the same rows."""
    m, wide = b.m, torch.zeros(4, 3 * HD)
    m.rope_rows(b.rope, wide[1:2, :HD], None, wide[1, :HD][None], None, ints(1), 1, 0, HD, stream=b.stream)
    rows = m.QkvRows.from_buffer_copy(b.reached[0][1][1])
    assert rows.q == rows.q_out and rows.q_stride == rows.q_out_stride == HD


def test_a_call_that_fails_after_planning(b, monkeypatch):
    """The library may have made the new plan before it refused the call: what is reused next has to hold the rows of either."""
    call(b, "prefill_plan_scored_tc")
    many = b.m.make_prefill_tiles([(0, 2 * N, 0, 0, 0, 0)])
    big = torch.zeros(2 * N, HEADS * HD)
    fine = b.m.check
    monkeypatch.setattr(b.m, "check", lambda status: (_ for _ in ()).throw(b.m.Error(1, "refused")))
    for name, change in (("prefill_attention_scored_tc", dict(tiles=many, q=big, out=big, score=b.m.Score())), ("prefill_plan_scored_tc", dict(tiles=many, score=b.m.Score()))):
        b.ws.plan_rows = N
        with pytest.raises(b.m.Error):
            call(b, name, **change)
        with pytest.raises(ValueError):
            call(b, "prefill_attention_scored_tc", reuse_plan=True)
    monkeypatch.setattr(b.m, "check", fine)
    call(b, "prefill_attention_scored_tc", reuse_plan=True, q=big, out=big, score=b.m.Score())
