"""The tensor checks of lcr_b200.paged without a device."""
import pytest

torch = pytest.importorskip("torch")

from lcr_b200 import _tensors, paged  # noqa: E402


def test_refusals_name_the_argument():
    with pytest.raises(ValueError, match="lengths: a contiguous int32 tensor.*got Int .3. .*on cpu"):
        _tensors.pointers(("lengths",), "i", torch.zeros(3, dtype=torch.int32), 3)
    with pytest.raises(ValueError, match="q: dense bf16 rows.*got list"):
        _tensors.pointers(("q",), "H", [1], 1)
    with pytest.raises(ValueError, match="keys: a bf16 pool"):
        paged.kv_view(torch.zeros(1, 1, 1, 64), torch.zeros(1, 1, 1, 64))
    with pytest.raises(TypeError):
        _tensors.pointers(("a",), "i", None)
    with pytest.raises(TypeError):
        _tensors.pointers()
    with pytest.raises(ValueError):
        paged.token_probs(torch.zeros(2, 5), torch.zeros(2, 5))
    with pytest.raises(ValueError):
        i = torch.zeros(4, dtype=torch.int32)
        paged.plan_step(i.view(2, 2), i, i, i, i, i, page_size=16, held_out=i, free_count_out=i, row_starts=i,
                        kv_lengths=i, positions=i, slots=i, row_sequence=i)
