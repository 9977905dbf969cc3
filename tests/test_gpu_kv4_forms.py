"""Attention over 4-bit pages: every kernel of the library, and the parts of long rows,
within the bounds derived in oracle/kv4.py (attend_bounds)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from kv4_cases import DIMS, held_call, row_tiles  # noqa: E402


@pytest.mark.parametrize("dim,group", DIMS)
def test_every_row_tile_with_shared_heads(dim, group):
    for tile, (least, most) in row_tiles(dim, group).items():
        for ratio in {least, most}:
            held_call("fp16", dim, group, 16, 1, ratio, [1, 130, 0, 17], [1, 1, 1, 1], seed=ratio, max_q=1)


@pytest.mark.parametrize("dim,group", DIMS)
def test_every_row_tile_with_several_tokens(dim, group):
    for tile, (least, most) in row_tiles(dim, group).items():
        held_call("bf16" if tile == 16 else "fp16", dim, group, 32, 2, 1, [most + 70, 300, 3], [most, least, 2], seed=most,
                  max_q=most)


@pytest.mark.parametrize("ratio,qs", [(16, [1, 1]), (7, [2, 3]), (1, [90, 9])])
def test_dims_256_in_groups_of_32_and_more_rows_than_8(ratio, qs):
    held_call("bf16", 256, 32, 16, 2, ratio, [140, 60], qs, seed=ratio)


@pytest.mark.parametrize("dim,group", [f for f in DIMS if f[0] < 256])
def test_prompt_chunks_of_every_form(dim, group):
    held_call("fp16", dim, group, 16, 2, 1, [300, 70, 133], [140, 70, 1], seed=dim + group)


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 128), (256, 64)])
@pytest.mark.parametrize("wide", [1.0, 0.0])  # 0: every weight is 1 / length
def test_no_part_of_a_long_row_is_lost(dim, group, wide):
    held_call("fp16", dim, group, 64, 1, 4, [9000, 1, 4000], [1, 1, 2], seed=8, max_q=2, wide=wide)


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 128)])
@pytest.mark.parametrize("wide", [1.0, 0.0])
def test_no_part_of_a_prompt_behind_a_long_prefix_is_lost(dim, group, wide):
    held_call("fp16", dim, group, 64, 1, 1, [6100, 2000], [70, 66], seed=3, wide=wide)


def test_single_tokens_beside_drafts_and_chunks():
    held_call("fp16", 128, 64, 16, 2, 4, [500, 33, 410, 90, 0, 260], [1, 5, 60, 1, 0, 16], seed=5)


@pytest.mark.parametrize("dim,group,ratio", [(64, 64, 100), (128, 32, 130), (256, 64, 71), (256, 32, 40)])
def test_more_query_heads_of_a_kv_head_than_a_tile_has_rows(dim, group, ratio):
    held_call("bf16", dim, group, 16, 1, ratio, [300, 17, 0, 140], [1, 1, 1, 2], seed=ratio)


@pytest.mark.parametrize("dim,group,ratio", [(64, 32, 4), (128, 32, 7), (128, 128, 20), (256, 128, 3)])
def test_a_batch_whose_requests_are_in_a_few_parts_each(dim, group, ratio):
    lens = [17 * i % 911 + 1 for i in range(1, 61)]
    held_call("fp16", dim, group, 32, 1, ratio, lens, [1] * len(lens), seed=ratio, max_q=1)
