"""The splits that the plan of decode over codes leaves room for: what the cut by lengths can
come to (256 of one sequence), however long the longest sequence is. Runs without a GPU."""
import pytest

import gemma_kv as gk


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
@pytest.mark.parametrize("batch", [2, 3, 24, 64])
def test_splits_of_a_batch_are_bounded(heads, dim, batch):
    config = gk.make_config(1, 1 << 16, 64, 1 << 14, 64, heads, dim, 0)
    for keys in (8192, 131072, 131073, 500_000, 1 << 20, 2**31 - 1):
        size, splits = gk.decode_split_plan_fp8(config, batch, keys)
        assert splits <= 256 and size * splits >= keys and size % 64 == 0
    # As ever up to there.
    assert gk.decode_split_plan_fp8(config, batch, 131072) == (512, 256)
