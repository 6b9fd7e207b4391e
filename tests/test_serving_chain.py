"""The serving calls together, as a decoder uses them: rotary positions, attention of drafted
trees over a paged cache, the accepted paths appended, attention weight gathered and the cache
evicted, step after step, against the same in 64 bits."""

import math

import pytest
import torch

import flash_attention_2_lab_b200 as fa
from cache_utils import LN, attention_64, lse_bound, make_cache, out_bound, score_error, slots_of
from parity_utils import read_status
from test_kv_cache import evict_64
from test_rotary import bound as rotary_bound
from test_rotary import turn

pytestmark = pytest.mark.gpu

B, HK, GROUP, DIM, PAGE, SLOTS = 3, 2, 2, 64, 16, 112
BUDGET, RECENT, SINKS, T = 48, 8, 2, 7


def drafted(g):
    """(parents, depth, mask, path, counts) of one step's trees and their accepted paths."""
    parents = (torch.rand(B, T, generator=g) * torch.arange(T)).long() - (torch.arange(T) == 0).long()
    depth = torch.zeros(B, T, dtype=torch.long)
    path, counts = torch.zeros(B, T, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        for t in range(1, T):
            depth[b, t] = depth[b, parents[b, t]] + 1
        way, t = [], int(torch.randint(0, T, (1,), generator=g))
        while t >= 0:
            way.append(t)
            t = int(parents[b, t])
        path[b, : len(way)] = torch.tensor(way[::-1], dtype=torch.int32)
        counts[b] = len(way)
    counts[1] = min(int(counts[1]), 1)
    return parents, depth, fa.tree_mask_from_parents(parents), path, counts


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_decoding_with_trees_and_eviction(layout):
    g = torch.Generator().manual_seed(31)
    k_pages, v_pages, table, _ = make_cache([0] * B, HK, DIM, PAGE, torch.float16, room=SLOTS)
    lengths = torch.zeros(B, dtype=torch.int32).cuda()
    seen = torch.zeros(B, dtype=torch.long)  # tokens so far: the next position
    weights = torch.zeros(B, HK, SLOTS).cuda()
    positions = torch.full((B, HK, SLOTS), -1, dtype=torch.int32).cuda()
    f, factor = fa.rotary_frequencies(DIM, scaling="linear", factor=2.0, device="cuda")
    scale = DIM ** -0.5

    def draw(heads, n):  # rows of a projection [B, N, H, D]
        return torch.randn(B, n, heads, DIM, generator=g).half().cuda().transpose(1, 2)

    # the prompts, of unequal length, in one chunk that attends to itself
    counts = torch.tensor([60, 33, 1], dtype=torch.int32)
    n = int(counts.max())
    q, k, v = draw(HK * GROUP, n), draw(HK, n), draw(HK, n)
    at = torch.arange(n).repeat(B, 1)
    q, k = fa.apply_rotary(q, k, at.cuda(), f, layout=layout, attention_factor=factor)
    out, lse = fa.tree_attention(q, k_pages, v_pages, table, lengths, k, v, tree_sizes=counts.cuda())
    for b in range(B):
        m = int(counts[b])
        ref = attention_64(q[b, :, :m].cpu(), k[b, :, :m].double().cpu(), v[b, :, :m].double().cpu(),
                           torch.ones(m, m, dtype=torch.bool).tril(), scale)
        assert ((out[b, :, :m].double().cpu() - ref[0]).abs()
                <= out_bound(ref[0], *ref[2:], torch.float16, DIM)).all()
    lengths = fa.append_to_cache(k, v, k_pages, v_pages, table, lengths, counts=counts.cuda(),
                                 weights=weights, positions=positions, new_positions=at.int().cuda())
    seen += counts
    fa.check_cache(k_pages, table, lengths)
    evictions = 0
    for step in range(6):
        parents, depth, mask, path, counts = drafted(g)
        at = seen[:, None] + depth
        raw_q, raw_k, v = draw(HK * GROUP, T), draw(HK, T), draw(HK, T)
        q, k = fa.apply_rotary(raw_q, raw_k, at.cuda(), f, layout=layout, attention_factor=factor)
        for x, y in ((raw_q, q), (raw_k, k)):
            ref = turn(x, at.cuda(), f, layout, factor)
            assert ((y.double() - ref).abs() <= rotary_bound(ref, x, torch.float16, factor)).all()
        out, lse = fa.tree_attention(q, k_pages, v_pages, table, lengths, k, v, tree_mask=mask.cuda())
        before = weights.clone()
        fa.accumulate_attention_weight(weights, q, k_pages, table, lengths, lse)
        ns = lengths.tolist()
        for b in range(B):
            kk = torch.cat([slots_of(k_pages, table, b, ns[b]), k[b].double()], 1).cpu()
            vv = torch.cat([slots_of(v_pages, table, b, ns[b]), v[b].double()], 1).cpu()
            sees = torch.cat([torch.ones(T, ns[b], dtype=torch.bool), mask[b]], 1)
            ref, ref_lse, spread, reach, size, count = attention_64(q[b].cpu(), kk, vv, sees, scale)
            err = (out[b].double().cpu() - ref).abs()
            assert (err <= out_bound(ref, spread, reach, size, count, torch.float16, DIM)).all()
            assert ((lse[b].double().cpu() - ref_lse).abs() <= lse_bound(ref_lse, size, count, DIM)).all()
            qq = q[b].double().cpu().unflatten(0, (HK, GROUP))
            s = torch.einsum("hgtd,hnd->hgtn", qq, kk[:, : ns[b]]) * scale
            p = torch.exp(s - lse[b].double().cpu().unflatten(0, (HK, GROUP))[..., None])
            mag = torch.einsum("hgtd,hnd->hgtn", qq.abs(), kk[:, : ns[b]].abs()) * scale + 20
            bound = (p * (score_error(mag, DIM) + (GROUP * T + 8) * LN)).sum((1, 2))
            want = before[b, :, : ns[b]].double().cpu() + p.sum((1, 2))
            assert ((weights[b, :, : ns[b]].double().cpu() - want).abs() <= bound + 2 * LN * want).all()
        # the accepted paths join the cache
        new = fa.append_to_cache(k, v, k_pages, v_pages, table, lengths, path=path.cuda(),
                                 counts=counts.cuda(), weights=weights, positions=positions,
                                 new_positions=at.int().cuda())
        for b in range(B):
            way = path[b, : int(counts[b])].long()
            assert torch.equal(slots_of(k_pages, table, b, int(new[b]))[:, ns[b]:], k[b, :, way.cuda()].double())
            assert positions[b, 0, ns[b]: int(new[b])].tolist() == at[b, way].tolist()
            assert (weights[b, :, ns[b]: int(new[b])] == 0).all()
        lengths, seen = new, seen + counts
        # and what weighed least leaves it
        ns = lengths.tolist()
        kept = [[evict_64(weights[b, h].tolist(), positions[b, h].tolist(), ns[b], BUDGET, RECENT, SINKS)
                 for h in range(HK)] for b in range(B)]
        old = [(slots_of(k_pages, table, b, ns[b]), slots_of(v_pages, table, b, ns[b])) for b in range(B)]
        old_w, old_p = weights, positions
        weights, positions, lengths = fa.evict_from_cache(k_pages, v_pages, table, lengths, weights, positions,
                                                          BUDGET, recent=RECENT, sinks=SINKS)
        for b in range(B):
            m = min(ns[b], BUDGET)
            evictions += ns[b] > BUDGET
            assert int(lengths[b]) == m
            for h in range(HK):
                src = kept[b][h]
                assert torch.equal(slots_of(k_pages, table, b, m)[h], old[b][0][h, src])
                assert torch.equal(slots_of(v_pages, table, b, m)[h], old[b][1][h, src])
                assert torch.equal(weights[b, h, :m], old_w[b, h, src])
                assert torch.equal(positions[b, h, :m], old_p[b, h, src])
                if ns[b] > BUDGET:  # the newest and the first are never among those that leave
                    there = set(positions[b, h, :m].tolist())
                    assert set(range(SINKS)) <= there
                    assert set(range(int(seen[b]) - RECENT, int(seen[b]))) <= there
    assert evictions >= 6 and read_status() == 0


def test_a_captured_step_replays():
    """A whole step in a graph: its lengths, weights and pages are state that every replay carries
    on, as running the calls again does."""
    g = torch.Generator().manual_seed(32)

    def state():
        k_pages, v_pages, table, lengths = make_cache([40, 50], HK, DIM, PAGE, torch.float16, room=20)
        slots = table.shape[1] * PAGE
        weights = torch.rand(2, HK, slots, generator=torch.Generator().manual_seed(33)).cuda()
        positions = torch.arange(slots).int().repeat(2, HK, 1).cuda()
        return [k_pages, v_pages, table, lengths, weights, positions, lengths.long()[:, None].clone()]

    q, k, v = (torch.randn(2, h, 1, DIM, generator=g).half().cuda() for h in (HK * GROUP, HK, HK))
    f, _ = fa.rotary_frequencies(DIM, device="cuda")

    def step(s):
        k_pages, v_pages, table, lengths, weights, positions, seen = s
        qr, kr = fa.apply_rotary(q, k, seen, f)
        out, lse = fa.tree_attention(qr, k_pages, v_pages, table, lengths, kr, v)
        fa.accumulate_attention_weight(weights, qr, k_pages, table, lengths, lse)
        longer = fa.append_to_cache(kr, v, k_pages, v_pages, table, lengths, weights=weights,
                                    positions=positions, new_positions=seen.int())
        w, p, n = fa.evict_from_cache(k_pages, v_pages, table, longer, weights, positions, 45, recent=4)
        weights.copy_(w)
        positions.copy_(p)
        lengths.copy_(n)
        seen.add_(1)
        return out

    eager, captured = state(), state()
    want = [step(eager).clone() for _ in range(5)]
    graph = torch.cuda.CUDAGraph()
    keep = [x.clone() for x in captured]
    with torch.cuda.graph(graph):
        out = step(captured)
    for x, y in zip(captured, keep):
        assert torch.equal(x.nan_to_num() if x.is_floating_point() else x,
                           y.nan_to_num() if y.is_floating_point() else y)
    for expected in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expected) and out.isfinite().all()
    for x, y in zip(captured[3:], eager[3:]):
        assert torch.equal(x, y)
    assert read_status() == 0 and not math.isnan(float(out.sum()))
