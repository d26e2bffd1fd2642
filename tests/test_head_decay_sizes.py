"""How many segments the linear attention's tokens are cut into, at the largest sizes that its operators take: no sum of 32 bits
passes their end, and what does not fit is refused.  Tensors on "meta" take no memory."""
import pytest
import torch

from transformer_b200.csrc import lib
from transformer_b200.parts import decay_attention

MOST = 2 ** 31 - 1


def test_counts_in_more_than_32_bits():
    assert lib.library().tb_head_decay_segments(MOST, 1, 64, 64) == MOST // 64 + 1
    assert lib.library().tb_head_decay_segments(MOST, MOST - MOST // 64, 64, 64) == MOST
    assert lib.library().tb_head_decay_segments(MOST, MOST - MOST // 64 + 1, 64, 64) < 0
    assert lib.library().tb_head_decay_segments(MOST, MOST, 64, 64) < 0


def test_scratch_in_more_than_32_bits():
    few, many = lib.head_decay_tc_work(MOST, 1, 64, 64), lib.head_decay_tc_work(MOST, MOST, 64, 64)
    assert 0 < few < many and many > (MOST + MOST // 256) * 64 * 64


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nt,B", [(MOST, MOST), (64 * 2 ** 20, MOST), (MOST, MOST - MOST // 64 + 1)])
def test_more_segments_than_32_bits_count(nt, B, dtype):
    z = lambda *s, dt=dtype: torch.empty(s, dtype=dt, device="meta")
    with pytest.raises(ValueError, match="segments"):
        decay_attention(z(nt, 1, 8), z(nt, 1, 8), z(nt, 1, 8), z(1, dt=torch.float32), z(B, 1, 8, 8, dt=torch.float32), z(B + 1, dt=torch.int32),
                        z(B, dt=torch.int32), z(nt, 1, 8))
