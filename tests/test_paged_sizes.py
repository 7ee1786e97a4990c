"""What the host computes for the paged operators' launches and workspaces, on the CPU."""

import pytest
import torch


def test_a_prompt_call_counts_the_tiles_that_run():
    """16 sequences of 32 rows of 4 heads a kv head are 16 tiles of 128 columns a kv head: 128 workgroups for 256 CUs, so the length is
    cut. One sequence of as many rows makes as many tiles; 32 sequences fill the chip."""
    from ssd import ops

    floats = lambda m, s: ops.paged_prompt_ws_floats(m, 32, 8, 128, s, 8192)  # noqa: E731
    four = 32 * 4 * 130  # floats a row: four parts
    assert floats(16 * 32, 16) == 16 * 32 * four and floats(512, 1) == 512 * four
    assert floats(15 * 32, 15) == 15 * 32 * four
    assert floats(32 * 32, 32) == 0 and floats(1024, 1) == 0


def test_prompt_workspaces_of_one_sequence_follow_from_its_tiles():
    from ssd import ops

    for m in (1, 7, 100, 333, 512):
        one = ops.paged_prompt_ws_floats(m, 32, 8, 128, 1, 16384)
        tiles = 8 * -(-m * 4 // 128)
        assert one == (0 if tiles >= 256 else m * 32 * min(512 // tiles, 32) * 130)
    assert ops.paged_prompt_ws_floats(0, 32, 8, 128, 4, 16384) == 0


@pytest.mark.parametrize("m,v,chunks", [(1, 128256, 16), (25, 128256, 16), (64, 128256, 16), (300, 128256, 4), (400, 128256, 1), (25, 50257, 7),
                                        (150, 50257, 1), (25, 32000, 1), (25, 200000, 25), (1, 1 << 24, 64), (0, 128256, 16)])
def test_token_logprobs_cut_rows_by_columns_whatever_their_type(m, v, chunks):
    """A thread takes 32 columns at a time; a chunk leaves a record of 32 bytes and 8 for each alternative."""
    from ssd import ops

    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        assert ops.token_logprobs_ws_bytes(m, v, dtype, 5) == (0 if chunks == 1 else m * chunks * (32 + 40))


def test_attention_workspaces_hold_scores_where_they_are_kept():
    """Scores [row][head][slots] up to 16 (row, head) pairs a kv head. 96 rows of 32 heads, 4032 slots in 8 groups of 512: 64 pairs."""
    from ssd import ops

    floats = lambda m, pairs: ops.paged_attn_ws_floats(m, 32, 128, 4032, 128, pairs)  # noqa: E731
    records, scores = 32 * 8 * 132, 32 * 4032  # a row's
    assert floats(96, 0) == 96 * 32 * 8 * 130
    assert floats(96, 1) == floats(96, True) == floats(96, 16) == 96 * (records + scores)
    assert floats(96, 17) == floats(96, 64) == max(96 * records, 16 * (records + scores))
    sizes = [floats(m, 64) for m in range(1, 97)]
    assert sizes == sorted(sizes)  # enough for fewer rows, whose call may keep its scores
    assert sizes[3] >= floats(4, 16)


def test_launches_whose_size_passes_64_bits_are_refused():
    from test_paged import BAD, RANGE, A, _batch, _kv, _refused

    most, ld = (1 << 31) - 1, 1 << 40
    wide = _batch(n_seq=1 << 30, rows_max=300, table_cols=1 << 24, ld_table=1 << 24)
    for kv in (1 << 30, most):
        c = _kv(kv_heads=kv)
        _refused("ssd_paged_write_bf16", (c, wide, A, ld, A, ld, most, None), RANGE, "workgroups")
        _refused("ssd_paged_read_bf16", (c, wide, most, A, ld, A, ld, None), RANGE, "workgroups")
        args = (A, ld, 1, kv, 1 << 30, 64, 0.1, A, (1 << 63) - 1, None, 0, 0, 1.0, A, ld, None)
        _refused("ssd_paged_attention_bf16", (c, wide, *args), RANGE, "workgroups")
        for layers in (1 << 20, 1 << 30):
            args = (A, most, most, 1 << 30, 1, 1, A + 4096, A, None)
            _refused("ssd_paged_evict", (c, layers, (1 << 63) - 1, wide, wide, *args), RANGE, "workgroups")
    # 2^20 rows of 2^15 heads in 2^22 groups: floats past 64 bits
    args = (A, ld, 1 << 20, 1 << 15, 1 << 30, 64, 0.1, A, 1 << 40, None, 0, 0, 1.0, A, ld, None)
    _refused("ssd_paged_attention_bf16", (_kv(head_dim=128), wide, *args), BAD, "workspace")


def test_weights_that_are_made_from_q_again_refuse_it_as_the_output():
    from test_paged import BAD, A, _batch, _kv, _refused

    args = (A, 256, 20, 4, 64, 64, 0.1, A, 1 << 20, A, 128, 64, 1.0, A, 256, None)
    _refused("ssd_paged_attention_bf16", (_kv(), _batch(rows_max=9), *args), BAD, "out must not be q")  # 18 pairs of a kv head
