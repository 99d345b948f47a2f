"""token_logprobs on rows shared by a cluster of blocks: the blocks write their sums and candidates into the first
block's shared memory, so they must know that it runs, also where a busy GPU starts a cluster's blocks late."""
import re
from pathlib import Path

import pytest
import torch


def test_blocks_meet_before_they_write_into_the_first_ones_memory():
    """In the source: a cluster-wide arrive before the pass and its wait before the first remote write."""
    text = (Path(__file__).resolve().parent.parent / "trifuse_b200" / "csrc" / "logprobs.cu").read_text()
    kernel = text[text.index("logprobs_kernel("):]
    arrive, wait = kernel.index("barrier.cluster.arrive"), kernel.index("barrier.cluster.wait")
    remote = re.search(r"\bto->\w+\[slice\]", kernel).start()
    assert arrive < kernel.index("auto fetch") < wait < remote < kernel.index("cluster.sync()")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dtype", [(1, torch.float32), (18, torch.bfloat16), (37, torch.float32), (74, torch.bfloat16)])
def test_clusters_on_a_busy_gpu(rows, dtype):
    """Clusters that find most SMs taken by other streams' blocks give the bits of a quiet GPU."""
    from trifuse_b200 import ops
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, 50304, generator=g) * 2.5).to(dtype).cuda()
    t = torch.randint(0, 50304, (rows,), generator=g).cuda()
    want = ops.token_logprobs(x, t, top=20)
    a = torch.randn(4096, 4096, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        with torch.cuda.stream(streams[0]):
            a @ a
        got = []
        for s in streams[1:]:
            with torch.cuda.stream(s):
                got.append(ops.token_logprobs(x, t, top=20))
        torch.cuda.synchronize()
        for r in got:
            for u, v in zip(want, r):
                assert torch.equal(u, v)
    assert ops.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V", [(3, 50304), (200, 50304), (200, 9001), (1, 250001)])
def test_expired_waits_are_told_and_do_no_harm(rows, V):
    """With a wait limit of one cycle a wait that its first try does not meet runs out and leaves the error code; the
    results are those of the whole rows all the same, since no slot is read or refilled before its copy has landed."""
    from trifuse_b200 import ops
    from trifuse_b200._lib import check, lib
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(rows, V, generator=g) * 2.5).cuda()
    t = torch.randint(0, V, (rows,), generator=g).cuda()
    want = ops.token_logprobs(x, t, top=20)
    assert ops.device_error() == 0
    check(lib().tf_set_wait_limit(1))
    try:
        got = ops.token_logprobs(x, t, top=20)
        assert ops.device_error() in (0, 72)
    finally:
        check(lib().tf_set_wait_limit(0))
    for u, v in zip(want, got):
        assert torch.equal(u, v)
    ops.token_logprobs(x, t, top=20)
    assert ops.device_error() == 0
