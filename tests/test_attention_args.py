"""What attention refuses beside tests/test_operator_args.py, without a GPU."""

import pytest

from raceline_amd import lib
from tests.test_operator_args import ATTN


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_a_scale_that_passes_fp32_in_base_2_is_refused(scale):
    """Scores are taken in base 2: scale times log2 e was infinite and every row NaN."""
    with pytest.raises(lib.RlqError, match="scale"):
        lib.call("rlq_attention", *{**ATTN, "scale": scale}.values())
