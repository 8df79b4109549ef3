"""The tensor checks of lcr_b200.paged without a device."""
import pytest

torch = pytest.importorskip("torch")

from lcr_b200 import paged  # noqa: E402


def test_refusals_name_the_argument():
    i = torch.zeros(4, dtype=torch.int32)
    pool = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    rows = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=r"logits|probs.*got Float \[2, 5\].*on cpu"):
        paged.token_probs(torch.zeros(2, 5), torch.zeros(2, 5))
    with pytest.raises(ValueError, match="block_tables: an int32 matrix.*got Int .2, 2. .*on cpu"):
        paged.plan_step(i.view(2, 2), i, i, i, i, i, page_size=16, held_out=i, free_count_out=i, row_starts=i,
                        kv_lengths=i, positions=i, slots=i, row_sequence=i)
    with pytest.raises(ValueError, match="keys: a bf16 pool.*on cpu"):
        paged.qk_norm_rope_kv(rows, pool, pool, rows, i, i, torch.zeros(32))
    with pytest.raises(ValueError, match="tokens: an int32 matrix.*got list"):
        paged.verify_drafts([1], i, torch.zeros(1, 5), i, i.view(2, 2), i, None, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="keys: a bf16 pool"):
        paged.chunk_attention(rows, rows, pool, pool, i.view(2, 2), i, i, scale=0.1, workspace=i)
