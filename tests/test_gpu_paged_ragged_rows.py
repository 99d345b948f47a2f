"""Attention whose rows end inside a warp of the tensor-core kernel: its tensor-memory loads and stores are the whole
warp's, so lanes without a row of their own stay with the others throughout."""
from pathlib import Path

import pytest
import torch

from tests.test_gpu_paged import BF16, F16, TYPES, run


def test_lanes_without_a_row_do_not_leave_their_warp():
    """In the source: the output loop, whose next turn loads tensor memory, brings the warp together at its end, and
    no lane skips ahead in it."""
    text = (Path(__file__).resolve().parent.parent / "trifuse_b200" / "csrc" / "paged_tile.cu").read_text()
    loop = text[text.index("for (int c = 0; c < D; c += 32) {", text.index("float* prow")):text.index("if (cleared) {")]
    assert "continue" not in loop and loop.rstrip().rstrip("}").rstrip().split("\n")[-1].strip().startswith("__syncwarp();")


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [17, 31, 33, 47, 65, 97, 127, 130, 161, 200, 225, 255, 300])
def test_rows_that_end_inside_a_warp(act, cache, D, n):
    """Whole results and cut ones (a long history), the same bits again."""
    from trifuse_b200 import ops
    for new, kv in (([n, n, n], [n, n + 100, 400]), ([n], [9000])):
        q, k, v, table, plan, got = run(ops, new, kv, 2, 2, D, 16, act, cache, seed=n)
        assert torch.equal(ops.paged_attention(q, k, v, table, plan), got)


@pytest.mark.gpu
@pytest.mark.parametrize("act", [F16, BF16])
def test_grouped_rows_that_end_inside_a_warp(act):
    from trifuse_b200 import ops
    run(ops, [5, 7, 19, 37, 41], [8011, 300, 19, 4000, 41], 14, 2, 64, 32, act, act)
