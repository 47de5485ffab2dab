"""Which tokens the selection keeps when more are infinitely heavy than it may keep."""
import pytest

from paged_fixture import load_b200

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_b200()


@pytest.mark.parametrize("keep,sinks,recent,heavy,want", [
    (5, 2, 9, [], [0, 1, 91, 92, 93]),          # sinks, then the recent tokens from their front
    (3, 4, 4, [], [0, 1, 2]),
    (5, 2, 2, [50, 60], [0, 1, 50, 60, 98]),    # infinite masses tie with protected tokens
    (6, 2, 2, [50, 60], [0, 1, 50, 60, 98, 99]),
    (4, 2, 2, [], [0, 1, 98, 99]),              # keep = sinks + recent: all of them, whatever the masses
    (120, 200, 200, [], list(range(100))),
])
def test_protected_tokens_that_do_not_fit(b, keep, sinks, recent, heavy, want):
    import torch
    mass = torch.rand(1, 100, device="cuda") * 1e30
    mass[0, heavy] = float("inf")
    one = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")
    d_keep, d_len = torch.empty(1, keep, dtype=torch.int32, device="cuda"), one(-1)
    b.evict_select(mass, one(100), one(0), 1, keep, sinks, recent, d_keep, d_len)
    assert d_len.item() == len(want) and d_keep[0, :len(want)].tolist() == want and (d_keep[0, len(want):] == -1).all()
