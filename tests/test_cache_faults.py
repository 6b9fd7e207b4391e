"""Calls that change a cache whose table, lengths or path lead outside it: what they leave out, and
that what they leave agrees with itself."""

import pytest
import torch

import flash_attention_2_lab_b200 as fa
from cache_utils import make_cache, slots_of
from parity_utils import read_status
from test_kv_cache import evict_64

pytestmark = pytest.mark.gpu

F16 = torch.float16
CACHE_BIT = 32


def slot_values(lengths, kv_heads, slots, seed):
    g = torch.Generator().manual_seed(seed)
    weights = torch.rand(len(lengths), kv_heads, slots, generator=g)
    positions = torch.stack([torch.stack([torch.randperm(slots, generator=g) for _ in range(kv_heads)])
                             for _ in lengths]).int()
    return weights.cuda(), positions.cuda()


@pytest.mark.parametrize("missing", [[3], [1], [0, 3], [1, 2, 3]])
@pytest.mark.parametrize("dim", [64, 128])
def test_evict_leaves_out_moves_of_missing_pages(dim, missing):
    read_status()
    page, budget = 16, 32
    lengths = [64, 50]
    k, v, table, ns = make_cache(lengths, 2, dim, page, F16, seed=3)
    weights, positions = slot_values(lengths, 2, 64, 4)
    bad = table.clone()
    bad[0, missing] = k.shape[0]
    k0, v0 = k.clone(), v.clone()
    w, p, n_new = fa.evict_from_cache(k, v, bad, ns, weights, positions, budget)
    assert read_status() == CACHE_BIT and n_new.tolist() == [budget, budget]
    left_out = 0
    for b, n in enumerate(lengths):
        for h in range(2):
            src = evict_64(weights[b, h].tolist(), positions[b, h].tolist(), n, budget, 0, 0)
            if b == 0:  # a move needs both pages
                stays = [to != come and (to // page in missing or come // page in missing)
                         for to, come in enumerate(src)]
                left_out += sum(stays)
                src = [to if s else come for to, (come, s) in enumerate(zip(src, stays))]
            assert torch.equal(w[b, h, :budget], weights[b, h, src])
            assert torch.equal(p[b, h, :budget], positions[b, h, src])
            assert (w[b, h, budget:] == 0).all() and (p[b, h, budget:] == -1).all()
            for x, x0 in ((k, k0), (v, v0)):  # the pages that are missing from the table hold what they held
                assert torch.equal(slots_of(x, table, b, budget)[h], slots_of(x0, table, b, n)[h, src])
    assert left_out > 0


def test_evict_holds_a_length_inside_the_table():
    read_status()
    lengths = [64, 50]
    k, v, table, ns = make_cache(lengths, 1, 64, 16, F16, seed=5)
    weights, positions = slot_values(lengths, 1, 64, 6)
    k, v = k.nan_to_num(), v.nan_to_num(posinf=2.0)
    k0 = k.clone()
    wrong = torch.tensor([-3, 65], dtype=torch.int32).cuda()
    w, p, n_new = fa.evict_from_cache(k, v, table, wrong, weights, positions, 32)
    assert read_status() == CACHE_BIT and n_new.tolist() == [0, 32]
    assert (w[0] == 0).all() and (p[0] == -1).all()
    src = evict_64(weights[1, 0].tolist(), positions[1, 0].tolist(), 64, 32, 0, 0)
    assert torch.equal(w[1, 0, :32], weights[1, 0, src])
    assert torch.equal(slots_of(k, table, 1, 32)[0], slots_of(k0, table, 1, 64)[0, src])
    assert torch.equal(slots_of(k, table, 0, 64), slots_of(k0, table, 0, 64))


@pytest.mark.parametrize("rows, dim", [(3, 64), (40, 128), (700, 64)])
@pytest.mark.parametrize("entry", [-1, "rows", 1 << 30])
@pytest.mark.parametrize("where", [0, 1, "last", "behind"])
def test_append_ends_before_a_bad_path_entry(where, entry, rows, dim):
    """Slots below the new length are written, the others keep what they held."""
    read_status()
    lengths = [20, 5]
    k, v, table, ns = make_cache(lengths, 2, dim, 16, F16, room=rows)
    k, v = k.nan_to_num(), v.nan_to_num(posinf=2.0)
    g = torch.Generator().manual_seed(8)
    key, value = (torch.randn(2, 2, rows, dim, generator=g).half().cuda() for _ in range(2))
    path = torch.randint(0, rows, (2, rows), generator=g).int()
    counts = torch.tensor([rows - 1, rows], dtype=torch.int32)
    at = {"last": rows - 2, "behind": rows - 1}.get(where, where)
    path[0, at] = rows if entry == "rows" else entry
    taken = [min(at, rows - 1), rows]  # an entry behind the count is not looked at
    slots = table.shape[1] * 16
    weights = torch.full((2, 2, slots), 7.0).cuda()
    positions = torch.full((2, 2, slots), 9, dtype=torch.int32).cuda()
    new = (1000 + torch.arange(rows, dtype=torch.int32)).repeat(2, 1).cuda()
    k0, v0 = k.clone(), v.clone()
    got = fa.append_to_cache(key, value, k, v, table, ns, path.cuda(), counts.cuda(), weights, positions, new)
    assert got.tolist() == [n + t for n, t in zip(lengths, taken)]
    assert read_status() == (0 if where == "behind" else CACHE_BIT)
    for b, n in enumerate(lengths):
        m, pick = n + taken[b], path[b, :taken[b]].long()
        for x, x0, rows_in in ((k, k0, key), (v, v0, value)):
            have, had = slots_of(x, table, b, slots), slots_of(x0, table, b, slots)
            assert torch.equal(have[:, n:m], rows_in[b][:, pick].double())
            assert torch.equal(have[:, :n], had[:, :n]) and torch.equal(have[:, m:], had[:, m:])
        assert (weights[b, :, n:m] == 0).all() and (weights[b, :, :n] == 7).all() and (weights[b, :, m:] == 7).all()
        assert (positions[b, :, n:m].cpu() == 1000 + pick.int()).all()
        assert (positions[b, :, :n] == 9).all() and (positions[b, :, m:] == 9).all()


def test_lengths_of_calls_without_rows_or_heads():
    """They are what the call would return with rows and heads: checked, counted and cut."""
    read_status()
    lengths = [20, 5, 31]
    k, v, table, ns = make_cache(lengths, 2, 64, 16, F16, room=1)
    none = torch.zeros(3, 2, 0, 64, dtype=F16).cuda()
    assert fa.append_to_cache(none, none, k, v, table, ns).tolist() == lengths
    zero = torch.zeros(3, dtype=torch.int32).cuda()
    assert fa.append_to_cache(none, none, k, v, table, ns, counts=zero).tolist() == lengths
    assert read_status() == 0
    assert fa.append_to_cache(none, none, k, v, table, ns, counts=zero + 2).tolist() == lengths
    assert read_status() == CACHE_BIT
    wrong = torch.tensor([-1, 33, 4], dtype=torch.int32).cuda()
    assert fa.append_to_cache(none, none, k, v, table, wrong).tolist() == [0, 32, 4]
    assert read_status() == CACHE_BIT
    # a cache without heads, as a shard may have
    k0, v0, rows = k[:, :0], v[:, :0], torch.zeros(3, 0, 4, 64, dtype=F16).cuda()
    counts = torch.tensor([4, 0, 1], dtype=torch.int32).cuda()
    assert fa.append_to_cache(rows, rows, k0, v0, table, ns, counts=counts).tolist() == [24, 5, 32]
    assert fa.append_to_cache(rows, rows, k0, v0, table, ns * 0).tolist() == [4, 4, 4]
    assert read_status() == 0
    assert fa.append_to_cache(rows, rows, k0, v0, table, ns).tolist() == [24, 9, 32]
    assert read_status() == CACHE_BIT
    weights, positions = torch.zeros(3, 0, 32).cuda(), torch.zeros(3, 0, 32, dtype=torch.int32).cuda()
    w, p, n = fa.evict_from_cache(k0, v0, table, ns, weights, positions, 18)
    assert w.shape == p.shape == (3, 0, 32) and n.tolist() == [18, 5, 18]
    assert read_status() == 0
