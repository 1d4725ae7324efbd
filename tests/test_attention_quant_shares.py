"""Into how many shares attention over codes cuts the keys of many query rows, seen from the workspace that it asks for: a host call, runs without a GPU."""
import pytest

from recurrent_drafting import _lib


def shares(B, new, keys, heads=32, kv=8):
    tokens = B * new
    need = _lib.load().rd_attention_quant_workspace_bytes(_lib.BF16, 8, tokens, B, heads, kv, 128, new, keys)
    return max(1, need // (tokens * heads * 132 * 4))  # fp32: an output of 128 features, its maximum and sum, in 16-byte pieces


@pytest.mark.parametrize("B, new, keys, fill", [(4, 128, 4096, 2), (2, 256, 4096, 2), (8, 64, 4096, 2), (2, 128, 8128, 4)])
def test_rows_that_are_alike_take_whole_rounds(B, new, keys, fill):
    """fill: the shares with which B rows of `new` tokens occupy two places on each of 148 multiprocessors, 296."""
    tiles = B * 8 * -(-new * 4 // 128)
    assert fill == 296 // tiles
    assert shares(B, new, keys) % fill == 0 and shares(B, new, keys) > fill


def test_one_row_and_short_ones():
    assert shares(1, 128, 4096) == 9  # 32 tiles of query rows
    assert shares(4, 128, 300) == 1 and shares(8, 128, 4000) == 1 and shares(4, 147, 2701) == 3
