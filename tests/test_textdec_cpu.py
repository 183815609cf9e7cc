"""TextDecoder's host-side choices, without a GPU: the buffers live on the CPU and no operator runs."""
import pytest
import torch


@pytest.mark.parametrize("max_tokens,block", [(100, 32), (128, 32), (1, 16)])
def test_every_position_has_a_row(lib, max_tokens, block):
    """A request holds whole blocks, so accepted rows may stand past max_tokens where that is no
    multiple of block; rows of a refused request stand past the last block (or at -1)."""
    from yolo11_cu_b200 import textdec
    dec = textdec.TextDecoder(2, rows=8, max_tokens=max_tokens, block=block, pool=16, device="cpu")
    holds = dec.max_blocks * block
    assert holds >= max_tokens
    pos = [-1, 0, max_tokens - 1, holds - 1, holds, holds + 500, 2 ** 31 - 1]
    dec.pos[:len(pos)] = torch.tensor(pos, dtype=torch.int32)
    rows = dec._places(len(pos))
    assert rows.shape == (len(pos), dec.width)
    assert dec.place.shape[0] == holds
    for i, p in enumerate(pos):
        assert torch.equal(rows[i], dec.place[min(max(p, 0), holds - 1)])
