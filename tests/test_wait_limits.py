"""Launches whose bounded waits run out, for every kernel with a pipeline of asynchronous copies.

With a limit of a nanosecond the first wait that is not over at once gives up.  The launch's output
is then invalid and the status word may say so, but its copies and products end before its blocks
do: the bit of a drain that ran out stays clear, and the launches that follow, which find the same
shared memory, are right.
"""

import pytest
import torch

from flash_attention_2_lab_b200 import _native
from parity_utils import abi_forward, read_status

pytestmark = pytest.mark.gpu

PRODUCER, PRODUCTS, SOFTMAX = 1, 2, 4  # status bits of waits that may run out here


def seeded(*shape, seed=0, dtype=torch.float16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def run_out(call):
    """`call` with waits that run out, between two ordinary ones with equal results."""
    lib = _native.lib()
    want = call()
    assert read_status() == 0
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    seen = 0
    try:
        lib.fa_set_wait_limit_ns(1)
        for _ in range(8):
            flush.zero_()  # the copies come from memory
            call()
            seen |= read_status()
    finally:
        lib.fa_set_wait_limit_ns(0)
    assert seen & ~(PRODUCER | PRODUCTS | SOFTMAX) == 0
    for _ in range(2):
        for a, b in zip(call(), want):
            assert torch.equal(a, b)
    assert read_status() == 0
    return seen


# a problem whose tiles all fit the ring, so that the producer itself never waits, and longer ones
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize(("b", "h", "n"), [(1, 2, 128), (1, 2, 256), (2, 3, 700), (8, 40, 1024)])
def test_forward(b, h, n, causal):
    q, k, v = (seeded(b, h, n, 64, seed=i) for i in range(3))
    run_out(lambda: [abi_forward(q, k, v, causal)])
