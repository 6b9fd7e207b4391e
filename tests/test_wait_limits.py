"""Launches whose bounded waits run out, for every kernel with a pipeline of asynchronous copies.

With a limit of a nanosecond a wait gives up that is not over when the hardware has looked at it
twice, some 14 us.  The launch's output is then invalid and the status word says so, but its copies
and products end before its blocks do: the bit of a drain that ran out stays clear, and the launches
that follow, which find the same shared memory, are right.
"""

import pytest
import torch

import flash_attention_2_lab_b200 as fa
from cache_utils import make_cache, roomy
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


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [20, 80])  # 80 and 320 rows: units of one and of two row tiles
@pytest.mark.parametrize("lengths", [[100, 128, 37], [5000, 0, 260]])
def test_tree_attention(lengths, tokens, dim):
    k, v, table, ns = make_cache(lengths, 2, dim, 16, torch.float16)
    rows = 4 * tokens
    table = roomy(table, 16, len(lengths) * 2 * rows)  # many rows go to the tiles
    q = seeded(len(lengths), 8, tokens, dim)
    kt, vt = (seeded(len(lengths), 2, tokens, dim, seed=i) for i in (1, 2))
    run_out(lambda: fa.tree_attention(q, k, v, table, ns, kt, vt))


def long_cache(dim):
    """448 heads of 4096 slots: a block has three parts of some 30 us, and the warp that brings the
    queries of a part waits for the end of an earlier one."""
    k, v = (torch.randn(56, 8, 4096, dim, generator=torch.Generator("cuda").manual_seed(i), device="cuda",
                        dtype=torch.float16) for i in range(2))
    return k, v, torch.arange(56, dtype=torch.int32).cuda()[:, None], torch.full((56,), 4096, dtype=torch.int32).cuda()


@pytest.mark.parametrize("tokens", [20, 40])
def test_tree_attention_that_gives_up(tokens):
    k, v, table, ns = long_cache(128)
    q = seeded(56, 32, tokens, 128)
    assert run_out(lambda: fa.tree_attention(q, k, v, table, ns)) & PRODUCER


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [100, 700])
def test_attention_weight(length, dim):
    k, _, table, ns = make_cache([length, 64, 0], 2, dim, 16, torch.float16)
    q, lse = seeded(3, 8, 20, dim), torch.full((3, 8, 20), 9.0).cuda()
    run_out(lambda: [fa.accumulate_attention_weight(torch.zeros(3, 2, table.shape[1] * 16).cuda(), q, k, table, ns,
                                                    lse)])


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_weight_that_gives_up(dim):
    k, _, table, ns = long_cache(dim)
    q, lse = seeded(56, 32, 32, dim), torch.full((56, 32, 32), 9.0).cuda()
    assert run_out(lambda: [fa.accumulate_attention_weight(torch.zeros(56, 8, 4096).cuda(), q, k, table, ns,
                                                           lse)]) & PRODUCER
