"""A workspace of another device is refused (its first field, the device, is changed for the call; no second GPU is needed)."""
import ctypes as C

import pytest

from paged_fixture import load_b200
from test_gpu_prefill_scored import Wave

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


def test_workspace_of_another_device(b):
    import torch
    w = Wave(b, torch, [(20, 0, 20, 0)], 2, 2, seed=5)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    ws, out, score = b.Workspace(64), torch.empty(20, 256, device="cuda"), b.Score()
    rope = b.Rope(rotary_dim=64)
    x = torch.randn(20, 256, device="cuda")
    q, k, v = (x.clone() for _ in range(3))
    pos, slots, one, zero = ints(*range(20)), ints(*[0] * 20), ints(20), ints(0)
    table = w.table.clone()
    lens = torch.full((1, 1), 20, dtype=torch.int32, device="cuda")
    mass, keep, count = torch.rand(1, 32, device="cuda"), torch.zeros(1, 8, dtype=torch.int32, device="cuda"), ints(8)
    b.prefill_plan_scored_tc(score, w.tiles, w.d_prefill, 16, ws)
    calls = {
        "rope_write_prefill_paged": lambda: b.rope_write_prefill_paged(w.layer, rope, q, k, v, q, pos, slots, pos, 2, ws),
        "rope_append_decode_batch_paged": lambda: b.rope_append_decode_batch_paged(w.layer, rope, q[:1], k[:1], v[:1], q[:1], zero, lens[0], ints(0), one, zero, 16, 2, ws),
        "attention_scored_batch_paged": lambda: b.attention_scored_batch_paged(w.layer, score, q, one, zero, one, zero, 1, 16, 2, out, ws),
        "attention_scored_ragged_paged": lambda: b.attention_scored_ragged_paged(w.layer, score, q, one, slots, pos, 20, 2, out, ws),
        "prefill_plan_scored_tc": lambda: b.prefill_plan_scored_tc(score, w.tiles, w.d_prefill, 16, ws),
        "prefill_attention_scored_tc": lambda: b.prefill_attention_scored_tc(w.layer, None, None, 0, score, q, w.d_prefill, w.tiles, 16, 2, out, ws, reuse_plan=True),
        "evict_select": lambda: b.evict_select(mass, one, zero, 1, 8, 0, 0, keep, count, ws),
        "evict_compact_paged_layers": lambda: b.evict_compact_paged_layers([w.layer], one, zero, 1, keep, count, None, ws),
        "evict_publish": lambda: b.evict_publish(table, zero, 1, keep, count, lens, one, 16, ws=ws),
    }
    device = C.cast(ws.h, C.POINTER(C.c_int))
    assert device[0] == torch.cuda.current_device()
    before = b.launch_count()
    for name, call in calls.items():
        device[0] += 1
        try:
            with pytest.raises(b.Error, match="another device"):
                call()
        finally:
            device[0] -= 1
    assert b.launch_count() == before
    for call in calls.values():
        call()
    assert ws.status() & b.STATUS_WAIT_TIMEOUT == 0  # (the ring append finds no ring in this table and says so)
