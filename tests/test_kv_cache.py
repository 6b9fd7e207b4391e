"""The paged cache's calls: refusals and helpers on the CPU; append, tree
attention, attention weight and eviction against 64 bits on the GPU."""

import math

import pytest
import torch

import flash_attention_2_lab_b200 as fa
from cache_utils import (LN, attention_64, lse_bound, make_cache, out_bound, roomy, score_error,
                         slots_of)
from flash_attention_2_lab_b200 import _native
from parity_utils import read_status

gpu = pytest.mark.gpu
CACHE_BIT = 32

F16, BF16 = torch.float16, torch.bfloat16


# ------------------------------------------------------------------ helpers (CPU)

def test_tree_mask_from_parents():
    mask = fa.tree_mask_from_parents(torch.tensor([-1, 0, 0, 2, 3, -1, 5]))
    up = {0: [], 1: [0], 2: [0], 3: [2, 0], 4: [3, 2, 0], 5: [], 6: [5]}
    for t in range(7):
        assert mask[t].nonzero().flatten().tolist() == sorted([t] + up[t])
    chain = fa.tree_mask_from_parents(torch.arange(-1, 69)[None].repeat(2, 1))
    assert torch.equal(chain, torch.ones(70, 70, dtype=torch.bool).tril().repeat(2, 1, 1))
    assert fa.tree_mask_from_parents(torch.tensor([-1])).tolist() == [[True]]
    assert fa.tree_mask_from_parents(torch.zeros(2, 0, dtype=torch.int32)).shape == (2, 0, 0)
    with pytest.raises(ValueError, match="parent must come before"):
        fa.tree_mask_from_parents(torch.tensor([0, 0]))


def test_check_cache_names_the_bad_entry():
    k, _, table, lengths = make_cache([5, 40], 1, 64, 16, F16, device="cpu")
    fa.check_cache(k, table, lengths)
    bad = table.clone()
    bad[1, 2] = k.shape[0]
    with pytest.raises(ValueError, match="sequence 1, entry 2"):
        fa.check_cache(k, bad, lengths)
    bad[1, 2] = -1
    with pytest.raises(ValueError, match="page -1 of sequence 1"):
        fa.check_cache(k, bad, lengths)
    bad = table.clone()
    bad[0, 1] = 999  # not used by a length of 5
    fa.check_cache(k, bad, lengths)
    for n in (-1, 49):
        with pytest.raises(ValueError, match="sequence 0"):
            fa.check_cache(k, table, torch.tensor([n, 3], dtype=torch.int32))


# ------------------------------------------------------------------ refusals (CPU)

def _cache_args(**change):
    a = dict(k_pages=torch.zeros(6, 2, 16, 64, dtype=F16), v_pages=torch.zeros(6, 2, 16, 64, dtype=F16),
             block_table=torch.zeros(3, 2, dtype=torch.int32), lengths=torch.zeros(3, dtype=torch.int32))
    a.update({k: v for k, v in change.items() if k in a})
    return a


CACHE_REFUSALS = [
    (dict(k_pages=torch.zeros(6, 2, 64, dtype=F16)), r"k_pages must have shape"),
    (dict(k_pages=torch.zeros(6, 2, 16, 64)), "k_pages must have dtype"),
    (dict(k_pages=torch.zeros(6, 2, 16, 80, dtype=F16)), "head dimension must be 64 or 128"),
    (dict(k_pages=torch.zeros(6, 2, 24, 64, dtype=F16)), "multiple of 16"),
    (dict(k_pages=torch.zeros(6, 2, 0, 64, dtype=F16)), "multiple of 16"),
    (dict(k_pages=torch.zeros(6, 16, 2, 64, dtype=F16).transpose(1, 2)), "k_pages must be contiguous"),
    (dict(block_table=torch.zeros(3, 2)), "block_table must have dtype torch.int32"),
    (dict(block_table=torch.zeros(6, dtype=torch.int32)), "block_table must have shape"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int32).t()), "block_table must have dense rows"),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), "lengths must have dtype torch.int32"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)), "lengths must have shape"),
    (dict(lengths=torch.zeros(6, dtype=torch.int32)[::2]), "lengths must be contiguous"),
]
V_REFUSALS = [
    (dict(v_pages=torch.zeros(5, 2, 16, 64, dtype=F16)), "identical shapes"),
    (dict(v_pages=torch.zeros(6, 2, 16, 64, dtype=BF16)), "same dtype"),
    (dict(v_pages=torch.zeros(6, 16, 2, 64, dtype=F16).transpose(1, 2)), "v_pages must be contiguous"),
]


def _tree(**change):
    a = dict(query=torch.zeros(3, 4, 5, 64, dtype=F16), k_tree=torch.zeros(3, 2, 5, 64, dtype=F16),
             v_tree=torch.zeros(3, 2, 5, 64, dtype=F16))
    cache = _cache_args(**change)
    a.update({k: v for k, v in change.items() if k not in cache})
    return fa.tree_attention(a.pop("query"), *cache.values(), **a)


@pytest.mark.parametrize(("change", "message"), CACHE_REFUSALS + V_REFUSALS + [
    (dict(query=torch.zeros(3, 4, 64, dtype=F16)), "query must have shape"),
    (dict(query=torch.zeros(2, 4, 5, 64, dtype=F16)), "query must have shape"),
    (dict(query=torch.zeros(3, 4, 5, 128, dtype=F16)), "query must have shape"),
    (dict(query=torch.zeros(3, 4, 5, 64, dtype=BF16)), "query must have the dtype of k_pages"),
    (dict(query=torch.zeros(3, 3, 5, 64, dtype=F16)), "multiple of the cache's heads"),
    (dict(v_tree=None), "k_tree and v_tree go together"),
    (dict(k_tree=torch.zeros(3, 2, 4, 64, dtype=F16)), "k_tree must have shape"),
    (dict(v_tree=torch.zeros(3, 1, 5, 64, dtype=F16)), "v_tree must have shape"),
    (dict(k_tree=None, v_tree=None, tree_mask=torch.ones(5, 5, dtype=torch.bool)), "tree_mask needs"),
    (dict(tree_mask=torch.ones(5, 5)), "tree_mask must have dtype torch.bool"),
    (dict(tree_mask=torch.ones(5, 4, dtype=torch.bool)), "tree_mask must have shape"),
    (dict(tree_mask=torch.ones(2, 5, 5, dtype=torch.bool)), "tree_mask must have shape"),
    (dict(tree_mask=torch.ones(3, 5, 5, dtype=torch.bool).transpose(1, 2)), "dense rows"),
    (dict(tree_sizes=torch.zeros(3)), "tree_sizes must have dtype"),
    (dict(tree_sizes=torch.zeros(2, dtype=torch.int32)), "tree_sizes must have shape"),
    (dict(), "query must be a CUDA tensor"),
])
def test_tree_attention_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _tree(**change)


def _append(**change):
    a = dict(key=torch.zeros(3, 2, 5, 64, dtype=F16), value=torch.zeros(3, 2, 5, 64, dtype=F16))
    cache = _cache_args(**change)
    a.update({k: v for k, v in change.items() if k not in cache})
    return fa.append_to_cache(a.pop("key"), a.pop("value"), *cache.values(), **a)


SLOTS = (3, 2, 32)


@pytest.mark.parametrize(("change", "message"), CACHE_REFUSALS + V_REFUSALS + [
    (dict(key=torch.zeros(3, 1, 5, 64, dtype=F16)), "key must have shape"),
    (dict(value=torch.zeros(3, 2, 4, 64, dtype=F16)), "value must have shape"),
    (dict(value=torch.zeros(3, 2, 5, 64, dtype=BF16)), "value must have the dtype"),
    (dict(path=torch.zeros(3, 4, dtype=torch.int32)), "path must have shape"),
    (dict(path=torch.zeros(3, 5)), "path must have dtype"),
    (dict(counts=torch.zeros(2, dtype=torch.int32)), "counts must have shape"),
    (dict(weights=torch.zeros(3, 2, 31)), "weights must have shape"),
    (dict(weights=torch.zeros(SLOTS, dtype=F16)), "weights must have dtype"),
    (dict(positions=torch.zeros(SLOTS, dtype=torch.int32)), "go together"),
    (dict(new_positions=torch.zeros(3, 5, dtype=torch.int32)), "go together"),
    (dict(positions=torch.zeros(SLOTS, dtype=torch.int32),
          new_positions=torch.zeros(3, dtype=torch.int32)), "new_positions must have shape"),
    (dict(path=torch.zeros(5, 3, dtype=torch.int32).t()), "must be contiguous"),
    (dict(), "k_pages must be a CUDA tensor"),
])
def test_append_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _append(**change)


def _evict(**change):
    a = dict(weights=torch.zeros(SLOTS), positions=torch.zeros(SLOTS, dtype=torch.int32), budget=8)
    cache = _cache_args(**change)
    a.update({k: v for k, v in change.items() if k not in cache})
    return fa.evict_from_cache(*cache.values(), **a)


@pytest.mark.parametrize(("change", "message"), CACHE_REFUSALS + V_REFUSALS + [
    (dict(weights=torch.zeros(3, 2, 33)), "weights must have shape"),
    (dict(weights=torch.zeros(3, 32, 2).transpose(1, 2)), "weights must be contiguous"),
    (dict(positions=torch.zeros(SLOTS)), "positions must have dtype"),
    (dict(budget=0), "budget must be positive"),
    (dict(recent=9), "the budget must hold both"),
    (dict(recent=5, sinks=4), "the budget must hold both"),
    (dict(recent=-1), "must not be negative"),
    (dict(), "k_pages must be a CUDA tensor"),
])
def test_evict_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _evict(**change)


def _weight(**change):
    a = dict(weights=torch.zeros(SLOTS), query=torch.zeros(3, 4, 5, 64, dtype=F16),
             lse=torch.zeros(3, 4, 5))
    cache = _cache_args(**change)
    a.update({k: v for k, v in change.items() if k not in cache})
    return fa.accumulate_attention_weight(a["weights"], a["query"], cache["k_pages"],
                                          cache["block_table"], cache["lengths"], a["lse"])


@pytest.mark.parametrize(("change", "message"), CACHE_REFUSALS + [
    (dict(weights=torch.zeros(3, 2, 16)), "weights must have shape"),
    (dict(query=torch.zeros(3, 5, 5, 64, dtype=F16)), "multiple of the cache's heads"),
    (dict(lse=torch.zeros(3, 4, 4)), "lse must be a contiguous float32"),
    (dict(lse=torch.zeros(3, 4, 5).double()), "lse must be a contiguous float32"),
    (dict(), "query must be a CUDA tensor"),
])
def test_weight_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _weight(**change)


def test_c_entries_refuse_without_gpu():
    import ctypes

    lib = _native.lib()

    def cache(k=4096, v=8192, table=4096, lengths=4096, stride=2, batch=3, heads=2, pages=6, size=16,
              per=2, dim=64):
        return ctypes.addressof(keep(
            (ctypes.c_int64 * 11)(k, v, table, lengths, stride, batch, heads, pages, size, per, dim)))

    kept = []

    def keep(x):
        kept.append(x)
        return x

    rows = ctypes.addressof(keep((ctypes.c_int64 * 4)(4096, 640, 320, 64)))
    odd = ctypes.addressof(keep((ctypes.c_int64 * 4)(4096, 640, 320, 60)))

    def append(c, k=rows, v=rows, n=5, out=1 << 20):
        return lib.fa_cache_append_sm100(c, k, v, n, None, None, None, None, None, out, None)

    def evict(c, budget=8, recent=0, sinks=0, w=4096, w2=8192, out=1 << 20, ws=4096, room=1 << 30):
        return lib.fa_cache_evict_sm100(c, w, 12288, w2, 16384, out, budget, recent, sinks, ws, room,
                                        None)

    def tree(c, q=rows, heads=4, tokens=5, kt=rows, vt=rows, mask=None, dtype=0, scale=0.125,
             out=4096, ws=4096, room=1 << 30):
        return lib.fa_tree_attention_sm100(c, q, heads, tokens, kt, vt, mask, 0, 5, None, dtype, scale,
                                           out, 4096, ws, room, None)

    def weight(c, q=rows, heads=4, tokens=5, lse=4096, w=4096, dtype=0, scale=0.125):
        return lib.fa_attention_weight_sm100(c, q, heads, tokens, lse, w, dtype, scale, None)

    for call in (append, evict, tree, weight):
        for kw, message in [(dict(size=8), "multiple of 16"), (dict(size=24), "multiple of 16"),
                            (dict(dim=96), "64 or 128"), (dict(batch=-1), "negative"),
                            (dict(k=4104), "aligned"), (dict(lengths=0), "null"),
                            (dict(table=0), "null"), (dict(k=0), "null"),
                            (dict(batch=70000), "too large"), (dict(per=1 << 30), "too large")]:
            assert call(cache(**kw)) == -1, (call, kw)
            assert message in _native.last_error(), (call, kw, _native.last_error())
        assert call(None) == -1 and "null" in _native.last_error()
        assert call(cache(batch=0)) == 0
    c = cache()
    for call, kw, message in [
        (append, dict(n=-1), "negative"), (append, dict(k=None), "null"), (append, dict(v=odd), "aligned"),
        (append, dict(out=None), "null"), (append, dict(out=4096), "in place"),
        (evict, dict(budget=0), "budget"), (evict, dict(recent=9), "budget"),
        (evict, dict(recent=5, sinks=4), "budget"), (evict, dict(ws=None), "null"),
        (evict, dict(w2=4096), "in place"), (evict, dict(out=4096), "in place"),
        (evict, dict(room=16), "workspace too small"), (evict, dict(ws=4112), "256-byte"),
        (tree, dict(heads=3), "multiple of the cache's heads"), (tree, dict(tokens=-1), "negative"),
        (tree, dict(dtype=2), "fp16 or bf16"), (tree, dict(scale=0.0), "scale"),
        (tree, dict(scale=math.inf), "scale"), (tree, dict(kt=None), "go together"),
        (tree, dict(kt=None, vt=None, mask=4096), "mask needs"), (tree, dict(q=odd), "query must be 16"),
        (tree, dict(vt=odd), "v_tree must be 16"), (tree, dict(out=None), "null"),
        (tree, dict(out=4104), "out must be 16"), (tree, dict(ws=4112), "256-byte"),
        (tree, dict(tokens=1 << 21), "too large"),
        (weight, dict(heads=3), "multiple"), (weight, dict(lse=None), "null"),
        (weight, dict(q=odd), "aligned"), (weight, dict(scale=math.nan), "scale"),
    ]:
        assert call(c, **kw) == -1, (call, kw)
        assert message in _native.last_error(), (call, kw, _native.last_error())


# ------------------------------------------------------------------ append (GPU)

APPENDS = [  # lengths, kv heads, new rows, page, dim
    ([0], 1, 1, 16, 64),
    ([0, 15, 16, 17, 31], 2, 3, 16, 64),
    ([5, 100], 3, 77, 32, 128),
    ([40, 0, 3], 1, 0, 16, 64),
    ([1] * 70, 2, 2, 48, 64),
]


@gpu
@pytest.mark.parametrize("with_path", [False, True])
@pytest.mark.parametrize(("dtype", "case"), [(F16, c) for c in APPENDS] + [(BF16, APPENDS[1])])
def test_append(case, dtype, with_path):
    lengths, hk, rows, page, dim = case
    g = torch.Generator().manual_seed(rows + dim)
    k, v, table, ns = make_cache(lengths, hk, dim, page, dtype, room=rows)
    key, value = (torch.randn(len(lengths), hk, rows, dim, generator=g).to(dtype).cuda() for _ in range(2))
    slots = table.shape[1] * page
    weights = torch.rand(len(lengths), hk, slots, generator=g).cuda()
    positions = torch.randint(0, 99, (len(lengths), hk, slots), generator=g).int().cuda()
    new_positions = torch.randint(100, 999, (len(lengths), rows), generator=g).int().cuda()
    path = counts = None
    if with_path:  # any rows, the same one twice among them
        path = torch.randint(0, max(rows, 1), (len(lengths), rows), generator=g).int().cuda()
        counts = torch.randint(0, rows + 1, (len(lengths),), generator=g).int().cuda()
    want = [t.clone() for t in (k, v, weights, positions)]
    new = []
    for b, n in enumerate(lengths):
        count = int(counts[b]) if with_path else rows
        new.append(n + count)
        for i in range(count):
            r, s = int(path[b, i]) if with_path else i, n + i
            at = (int(table[b, s // page]), slice(None), s % page)
            want[0][at], want[1][at] = key[b, :, r], value[b, :, r]
            want[2][b, :, s], want[3][b, :, s] = 0.0, int(new_positions[b, r])
    got = fa.append_to_cache(key, value, k, v, table, ns, path=path, counts=counts, weights=weights,
                             positions=positions, new_positions=new_positions)
    assert got.tolist() == new and got.dtype == torch.int32 and ns.tolist() == list(lengths)
    for x, y in zip((k, v, weights, positions), want):
        assert torch.equal(x.view(torch.int16 if x.dtype in (F16, BF16) else x.dtype),
                           y.view(torch.int16 if y.dtype in (F16, BF16) else y.dtype))
    assert read_status() == 0


@gpu
def test_append_of_strided_and_unaligned_rows():
    g = torch.Generator().manual_seed(7)
    k, v, table, ns = make_cache([3, 20], 2, 64, 16, F16, room=6)
    kv = torch.randn(2, 6, 2, 2, 64, generator=g).half().cuda()  # [B, N, k or v, H, D]
    odd = torch.randn(2, 2, 6, 67, generator=g).half().cuda()[..., 3:]
    for key, value in ((kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)), (odd, odd),
                       (odd[:1].expand(2, 2, 6, 64), odd[:, :1].expand(2, 2, 6, 64))):
        fa.append_to_cache(key, value, k, v, table, ns)
        for b, n in enumerate([3, 20]):
            assert torch.equal(slots_of(k, table, b, n + 6)[:, n:], key[b].double())
            assert torch.equal(slots_of(v, table, b, n + 6)[:, n:], value[b].double())


# ------------------------------------------------------------------ tree attention (GPU)

def reference(q, k, v, table, lengths, kt, vt, mask, sizes, scale):
    """attention_64 of every sequence, stacked."""
    got = []
    t = q.shape[2]
    for b, n in enumerate(lengths):
        kk, vv = slots_of(k, table, b, n).cpu(), slots_of(v, table, b, n).cpu()
        size = t if sizes is None else int(sizes[b])
        there = torch.arange(t) < size
        seen = there[:, None].expand(t, n)
        if kt is not None:
            kk = torch.cat([kk, kt[b].double().cpu()], 1)
            vv = torch.cat([vv, vt[b].double().cpu()], 1)
            tree = (torch.ones(t, t, dtype=torch.bool).tril() if mask is None
                    else (mask if mask.dim() == 2 else mask[b]).cpu())
            seen = torch.cat([seen, tree & there[:, None] & there], 1)
        got.append(attention_64(q[b].cpu(), kk, vv, seen, scale))
    return [torch.stack(x) for x in zip(*got)]


def check_attention(got, want, dtype, dim):
    (out, lse), (ref, ref_lse, spread, reach, size, count) = got, want
    assert out.dtype == dtype and out.is_contiguous() and lse.dtype == torch.float32
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(lse == -math.inf, ref_lse == -math.inf)
    some = ref_lse != -math.inf
    assert ((out - ref).abs() <= out_bound(ref, spread, reach, size, count, dtype, dim)).all()
    assert (out[~some] == 0).all()
    assert ((lse - ref_lse).abs() <= lse_bound(ref_lse, size, count, dim))[some].all()


TREES = [  # lengths, kv heads, group, tokens, page
    ([1], 1, 1, 1, 16),
    ([0], 1, 1, 1, 16),
    ([0, 1, 15, 16, 17, 63, 64, 65], 1, 2, 1, 16),
    ([130, 7], 2, 4, 1, 16),
    ([300, 0, 37], 2, 3, 5, 32),      # 15 rows
    ([200, 64], 1, 1, 16, 64),        # exactly a row tile
    ([100, 129], 2, 1, 17, 48),       # one row more
    ([77], 1, 8, 4, 16),              # two row tiles of 16
    ([257], 1, 8, 13, 16),            # 104 rows
    ([90, 200], 2, 2, 70, 32),        # 140 rows, a tree longer than a tile of keys
    ([500], 1, 1, 129, 16),
    ([0, 0], 2, 2, 33, 16),           # the tree alone
]


# with room for few slots, and for so many that many rows go to the tensor-core tiles
ROOM = pytest.mark.parametrize("room", ["tight", "roomy"])


def table_of(table, room, page, rows):
    return roomy(table, page, rows) if room == "roomy" else table


@gpu
@ROOM
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", TREES)
def test_tree_attention(case, dtype, dim, room):
    lengths, hk, group, t, page = case
    g = torch.Generator().manual_seed(sum(lengths) + t)
    k, v, table, ns = make_cache(lengths, hk, dim, page, dtype)
    table = table_of(table, room, page, len(lengths) * hk * group * t)
    q = (1.5 * torch.randn(len(lengths), hk * group, t, dim, generator=g)).to(dtype).cuda()
    kt, vt = (torch.randn(len(lengths), hk, t, dim, generator=g).to(dtype).cuda() for _ in range(2))
    parents = (torch.rand(len(lengths), t, generator=g) * torch.arange(t)).long() - (torch.arange(t) == 0).long()
    mask = fa.tree_mask_from_parents(parents).cuda()
    scale = dim ** -0.5
    for tree in ((kt, vt, mask), (kt, vt, None), (None, None, None)):
        got = fa.tree_attention(q, k, v, table, ns, *tree)
        check_attention(got, reference(q, k, v, table, lengths, *tree, None, scale), dtype, dim)
    assert read_status() == 0


@gpu
@ROOM
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_see_nothing_and_padding(dim, room):
    """Empty mask rows over an empty cache; sequences with fewer tokens than the batch, or none."""
    g = torch.Generator().manual_seed(9)
    lengths, hk, group, t = [0, 40, 0, 21, 30], 2, 2, 20
    k, v, table, ns = make_cache(lengths, hk, dim, 16, F16)
    table = table_of(table, room, 16, 5 * 4 * t)
    q = torch.randn(5, 4, t, dim, generator=g).half().cuda()
    kt, vt = (torch.randn(5, hk, t, dim, generator=g).half().cuda() for _ in range(2))
    mask = torch.rand(t, t, generator=g).cuda() < 0.3
    mask[3] = False
    mask[0] = False
    sizes = torch.tensor([t, 7, 5, 0, 1], dtype=torch.int32).cuda()
    for rows in (torch.arange(5), torch.arange(7, t)):  # padding may hold anything
        for x in (q, kt, vt):
            for b in range(1, 5):
                x[b, :, max(int(sizes[b]), int(rows[0])):] = math.nan
    got = fa.tree_attention(q, k, v, table, ns, kt, vt, tree_mask=mask, tree_sizes=sizes, scale=0.3)
    want = reference(q.nan_to_num(), k, v, table, lengths, kt, vt, mask, sizes, 0.3)
    check_attention(got, want, F16, dim)
    assert (got[1][0, :, [0, 3]] == -math.inf).all() and (got[1][3] == -math.inf).all()


LONG = [  # lengths, kv heads, group, tokens, page: parts of units over many blocks
    ([5000, 130, 0], 1, 2, 50, 16),    # 100 rows
    ([3000, 4097], 2, 1, 20, 48),
    ([4100], 1, 5, 52, 128),           # 260 rows: a second pair of row tiles
    ([2500, 77, 1300], 2, 3, 45, 32),  # 135 rows
    ([6000, 5], 1, 4, 4, 64),          # 16 rows
]


@gpu
@ROOM
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", LONG)
def test_long_caches_and_many_rows(case, dim, room):
    lengths, hk, group, t, page = case
    dtype = BF16 if page == 48 else F16
    g = torch.Generator().manual_seed(sum(lengths) + t)
    k, v, table, ns = make_cache(lengths, hk, dim, page, dtype)
    table = table_of(table, room, page, len(lengths) * hk * group * t)
    q = (1.5 * torch.randn(len(lengths), hk * group, t, dim, generator=g)).to(dtype).cuda()
    kt, vt = (torch.randn(len(lengths), hk, t, dim, generator=g).to(dtype).cuda() for _ in range(2))
    sizes = torch.tensor([max(1, t - 7 * b) for b in range(len(lengths))], dtype=torch.int32)
    got = fa.tree_attention(q, k, v, table, ns, kt, vt, tree_sizes=sizes.cuda())
    check_attention(got, reference(q, k, v, table, lengths, kt, vt, None, sizes, dim ** -0.5), dtype, dim)
    assert read_status() == 0


@gpu
@ROOM
@pytest.mark.parametrize("t", [6, 20, 70])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinities_reach_only_the_rows_that_see_them(dtype, dim, t, room):
    g = torch.Generator().manual_seed(10)
    lengths = [50, 0]
    k, v, table, ns = make_cache(lengths, 1, dim, 16, dtype)
    table = table_of(table, room, 16, 2 * 3 * t)
    q = torch.randn(2, 3, t, dim, generator=g).to(dtype).cuda()
    kt, vt = (torch.randn(2, 1, t, dim, generator=g).to(dtype).cuda() for _ in range(2))
    mask = torch.ones(t, t, dtype=torch.bool).tril()
    mask[4, 2] = mask[5, 1] = mask[5, 3] = False
    clean = fa.tree_attention(q, k, v, table, ns, kt, vt, tree_mask=mask.cuda())
    vt[:, :, 2, 5] = math.inf
    vt[:, :, 3, 7] = math.nan
    kt[:, :, 1] = math.nan
    out, lse = fa.tree_attention(q, k, v, table, ns, kt, vt, tree_mask=mask.cuda())
    sees = mask.cuda()
    hit = sees[:, 1]  # a NaN key makes its row NaN
    assert out[:, :, hit].isnan().all() and lse[:, :, hit].isnan().all()
    check = ~hit
    assert torch.equal(lse[:, :, check], clean[1][:, :, check])
    wide = (~sees[:, 2] & ~sees[:, 3] & check).nonzero().flatten()
    assert len(wide)
    step = torch.finfo(dtype).eps
    # the step is then summed in another order and with P unrounded
    spread = 3 * step
    for row in wide.tolist():
        assert out[:, :, row].isfinite().all()
        assert ((out[:, :, row] - clean[0][:, :, row]).abs() <= spread * 4).all()
    # row 5 sees value 2 (infinite in element 5) and not value 3
    if not hit[5]:
        assert (out[:, :, 5, 5] == math.inf).all()
        assert out[:, :, 5, :5].isfinite().all() and out[:, :, 5, 6:].isfinite().all()


def _tall_tree(dtype, dim, room, seed):
    """A tree of 200 nodes, two tiles of keys, over a short cache, a long one, whose units lie in
    several parts, and none; most rows of either tile see some of nodes 2, 60, 150 and 199 and not
    others, and some see none of them."""
    g = torch.Generator().manual_seed(seed)
    lengths, t = [50, 3000, 0], 200
    k, v, table, ns = make_cache(lengths, 1, dim, 16, dtype)
    table = table_of(table, room, 16, 3 * 2 * t)
    q = torch.randn(3, 2, t, dim, generator=g).to(dtype).cuda()
    kt, vt = (torch.randn(3, 1, t, dim, generator=g).to(dtype).cuda() for _ in range(2))
    mask = torch.rand(t, t, generator=g) < 0.5
    mask[::5, [2, 60, 150, 199]] = False
    return lengths, k, v, table, ns, q, kt, vt, mask


@gpu
@ROOM
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_odd_values_in_every_tile_of_a_tree(dtype, dim, room):
    lengths, k, v, table, ns, q, kt, vt, mask = _tall_tree(dtype, dim, room, 24)
    clean = fa.tree_attention(q, k, v, table, ns, kt, vt, tree_mask=mask.cuda())
    for node, element, value in ((2, 5, math.inf), (60, 7, math.nan), (150, 9, -math.inf), (199, 11, math.nan)):
        vt[:, :, node, element] = value
    out, lse = fa.tree_attention(q, k, v, table, ns, kt, vt, tree_mask=mask.cuda())
    assert torch.equal(lse, clean[1])
    ref, ref_lse, spread, reach, size, count = reference(q, k, v, table, lengths, kt, vt, mask, None, dim ** -0.5)
    out = out.cpu().double()
    fine = ref.isfinite()
    assert (~fine).any(2).any(2).all() and fine.all(-1)[:, :, ::5].all()
    assert torch.equal(out.nan_to_num(-7, 8, -8)[~fine], ref.nan_to_num(-7, 8, -8)[~fine])
    bound = out_bound(ref, spread, reach, size, count, dtype, dim)
    assert ((out - ref).abs() <= bound)[fine].all()
    assert read_status() == 0


@gpu
@ROOM
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("node", [2, 150])
def test_a_key_of_nan_reaches_only_the_rows_that_see_it(node, dim, room):
    lengths, k, v, table, ns, q, kt, vt, mask = _tall_tree(F16, dim, room, 25)
    clean = fa.tree_attention(q, k, v, table, ns, kt, vt, tree_mask=mask.cuda())
    kt[:, :, node] = math.nan
    got = fa.tree_attention(q, k, v, table, ns, kt, vt, tree_mask=mask.cuda())
    sees = mask[:, node].cuda()
    for x, y in zip(got, clean):
        assert x[:, :, sees].isnan().all() and torch.equal(x[:, :, ~sees], y[:, :, ~sees])


@gpu
@ROOM
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_of_every_size(dim, room):
    """Large scores, where the running maximum moves, and rows of equal ones."""
    g = torch.Generator().manual_seed(11)
    k, v, table, ns = make_cache([1400], 1, dim, 16, F16)
    table = table_of(table, room, 16, 80)
    q = torch.cat([30 * torch.randn(1, 2, 35, dim, generator=g), torch.zeros(1, 2, 5, dim)], 2).half().cuda()
    got = fa.tree_attention(q, k, v, table, ns, scale=0.125)
    check_attention(got, reference(q, k, v, table, [1400], None, None, None, None, 0.125), F16, dim)


@gpu
@ROOM
def test_strides_and_alignment_of_the_tree(room):
    g = torch.Generator().manual_seed(12)
    lengths = [33, 80]
    k, v, table, ns = make_cache(lengths, 2, 64, 16, F16)
    wide = table.new_zeros(2, table.shape[1] + 3)
    wide[:, : table.shape[1]] = table
    table_view = table_of(wide[:, : table.shape[1]], room, 16, 2 * 4 * 9)
    qkv = torch.randn(2, 9, 8, 64, generator=g).half().cuda()  # [B, T, heads of q, k and v, D]
    q, kt, vt = (qkv[:, :, a:b].transpose(1, 2) for a, b in ((0, 4), (4, 6), (6, 8)))
    odd = torch.randn(2, 4, 9, 65, generator=g).half().cuda()
    mask = (torch.rand(2, 9, 12, generator=g) < 0.5).cuda()[..., 2:11]
    for qq, kk, vv in ((q, kt, vt), (odd[..., 1:], odd[:, :2, :, :64], kt.expand(2, 2, 9, 64))):
        got = fa.tree_attention(qq, k, v, table_view, ns, kk, vv, tree_mask=mask)
        check_attention(got, reference(qq, k, v, table, lengths, kk, vv, mask, None, 0.125), F16, 64)


@gpu
def test_contiguous_cache_and_shared_pages():
    """One tensor [B, H_kv, capacity, D] as a cache; two sequences that share their first page."""
    g = torch.Generator().manual_seed(13)
    k, v = (torch.randn(3, 2, 112, 64, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(3, 4, 1, 64, generator=g).half().cuda()
    lengths = [112, 5, 50]
    table = torch.arange(3).int().cuda()[:, None]
    ns = torch.tensor(lengths, dtype=torch.int32).cuda()
    got = fa.tree_attention(q, k, v, table, ns)
    check_attention(got, reference(q, k, v, table, lengths, None, None, None, None, 0.125), F16, 64)
    k, v = (x.reshape(3, 2, 7, 16, 64).transpose(1, 2).reshape(21, 2, 16, 64).contiguous() for x in (k, v))
    table = torch.tensor([[4, 5], [4, 9], [4, 4]]).int().cuda()
    lengths = [20, 32, 31]
    ns = torch.tensor(lengths, dtype=torch.int32).cuda()
    got = fa.tree_attention(q, k, v, table, ns)
    check_attention(got, reference(q, k, v, table, lengths, None, None, None, None, 0.125), F16, 64)


@gpu
def test_many_sequences_and_one_long_one():
    """More sequences than threads of a block lay out at once, most of them empty or short."""
    lengths = [0, 1, 2, 40] * 40 + [3000] + [5] * 9
    g = torch.Generator().manual_seed(14)
    k, v, table, ns = make_cache([3000], 1, 64, 16, F16, spare=0)
    table = table.repeat(len(lengths), 1)
    ns = torch.tensor(lengths, dtype=torch.int32).cuda()
    q = torch.randn(len(lengths), 2, 1, 64, generator=g).half().cuda()
    got = fa.tree_attention(q, k, v, table, ns)
    want = reference(q, k, v, table[:1].repeat(len(lengths), 1), lengths, None, None, None, None, 0.125)
    check_attention(got, want, F16, 64)


@gpu
@pytest.mark.parametrize("batch, heads, t, dim", [(1100, 2, 1, 64), (1100, 2, 1, 128), (150, 16, 5, 64),
                                                  (150, 8, 5, 128)])
def test_more_units_than_blocks(batch, heads, t, dim):
    """Units that lie whole in a block among others, and the few that a cut goes through."""
    lengths = [[0, 1, 16, 40, 130, 161, 7][i % 7] for i in range(batch)]
    g = torch.Generator().manual_seed(23)
    k, v, one, _ = make_cache([161], 2, dim, 16, F16, spare=0, seed=23)
    k, v = k.nan_to_num_(nan=0.5), v.nan_to_num_(posinf=0.25)
    table = one.repeat(batch, 1)
    ns = torch.tensor(lengths, dtype=torch.int32).cuda()
    q = torch.randn(batch, heads, t, dim, generator=g).half().cuda()
    kt, vt = (torch.randn(batch, 2, t, dim, generator=g).half().cuda() for _ in range(2))
    sizes = torch.tensor([[t, 1, 0][i % 3] for i in range(batch)], dtype=torch.int32).cuda()
    room = roomy(table, 16, batch * heads * t) if t > 1 else table
    got = fa.tree_attention(q, k, v, room, ns, kt, vt, tree_sizes=sizes)
    want = reference(q, k.cpu(), v.cpu(), table.cpu(), lengths, kt, vt, None, sizes, dim ** -0.5)
    check_attention(got, want, F16, dim)


@gpu
def test_changes_in_place_are_seen_by_autograd():
    k, v, table, ns = make_cache([20, 5], 2, 64, 16, F16, room=8)
    weights = torch.zeros(2, 2, 32).cuda()
    positions = torch.zeros(2, 2, 32, dtype=torch.int32).cuda()
    state = (k, v, weights, positions)

    def counts():
        return [x._version for x in state]

    before = counts()
    rows = torch.zeros(2, 2, 3, 64, dtype=F16).cuda()
    fa.append_to_cache(rows, rows, k, v, table, ns, None, None, weights, positions,
                       torch.zeros(2, 3, dtype=torch.int32).cuda())
    assert all(a > b for a, b in zip(counts(), before))
    before = counts()
    fa.accumulate_attention_weight(weights, rows, k, table, ns, torch.zeros(2, 2, 3).cuda())
    assert [a > b for a, b in zip(counts(), before)] == [False, False, True, False]
    before = counts()
    fa.evict_from_cache(k, v, table, ns, weights, positions, 4)
    assert [a > b for a, b in zip(counts(), before)] == [True, True, False, False]


@gpu
@ROOM
@pytest.mark.parametrize("t", [3, 12, 50])
def test_same_bits_every_time_two_streams_and_a_graph(t, room):
    g = torch.Generator().manual_seed(15)
    lengths = [700, 33, 1500]
    k, v, table, ns = make_cache(lengths, 2, 64, 16, F16)
    table = table_of(table, room, 16, 3 * 8 * t)
    q = torch.randn(3, 8, t, 64, generator=g).half().cuda()
    kt, vt = (torch.randn(3, 2, t, 64, generator=g).half().cuda() for _ in range(2))
    first = fa.tree_attention(q, k, v, table, ns, kt, vt)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):
        for s in sides:
            with torch.cuda.stream(s):
                outs.append(fa.tree_attention(q, k, v, table, ns, kt, vt))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], first[0]) and torch.equal(o[1], first[1])
    graphs, held = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(fa.tree_attention(q, k, v, table, ns, kt, vt))
        graphs.append(graph)
    ns.copy_(torch.tensor([100, 1504, 7], dtype=torch.int32))  # lengths are read when it runs
    k.nan_to_num_(nan=0.25)
    v.nan_to_num_(posinf=0.5)
    want = fa.tree_attention(q, k, v, table, ns, kt, vt)
    for s, graph in zip(sides, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for o in held:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


@gpu
def test_empty_calls():
    k, v, table, ns = make_cache([3], 1, 64, 16, F16)
    for shape in ((1, 2, 0, 64), (1, 0, 4, 64)):
        out, lse = fa.tree_attention(torch.zeros(shape, dtype=F16).cuda(), k, v, table, ns)
        assert out.shape == shape and lse.shape == shape[:3]
    out, lse = fa.tree_attention(torch.zeros(0, 2, 1, 64, dtype=F16).cuda(), k, v, table[:0], ns[:0])
    assert out.shape == (0, 2, 1, 64)
    # no pages at all: every query sees nothing
    out, lse = fa.tree_attention(torch.zeros(1, 2, 1, 64, dtype=F16).cuda(), k[:0], v[:0], table[:, :0],
                                 ns * 0)
    assert (out == 0).all() and (lse == -math.inf).all()


# ------------------------------------------------------------------ attention weight (GPU)

WEIGHTS = [  # lengths, kv heads, group, tokens, page
    ([1], 1, 1, 1, 16),
    ([0, 1, 31, 32, 33, 255, 256, 257], 1, 2, 1, 16),
    ([300, 0, 37], 2, 4, 3, 32),
    ([130], 1, 7, 9, 48),      # 63 rows
    ([70, 300], 2, 8, 8, 16),  # 64 rows
    ([100], 1, 5, 13, 16),     # 65 rows: a second chunk
    ([40], 2, 4, 50, 16),      # 200 rows
    ([300, 1000], 1, 8, 81, 32),  # 648 rows: more than one pass over the keys
    ([5000, 3, 129], 3, 2, 2, 16),
    ([200] * 40, 4, 1, 1, 112),
]


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", WEIGHTS)
def test_attention_weight(case, dtype, dim):
    lengths, hk, group, t, page = case
    g = torch.Generator().manual_seed(sum(lengths) + t)
    k, v, table, ns = make_cache(lengths, hk, dim, page, dtype)
    q = (1.5 * torch.randn(len(lengths), hk * group, t, dim, generator=g)).to(dtype).cuda()
    _, lse = fa.tree_attention(q, k, v, table, ns)
    if t > 2:
        lse[:, :, 1] = -math.inf  # a row that saw nothing
    weights = torch.rand(len(lengths), hk, table.shape[1] * page, generator=g).cuda()
    before = weights.clone()
    for scale in (None, 0.07):
        weights.copy_(before)
        got = fa.accumulate_attention_weight(weights, q, k, table, ns, lse, scale=scale)
        assert got.data_ptr() == weights.data_ptr()
        sc = dim ** -0.5 if scale is None else scale
        for b, n in enumerate(lengths):
            kk = slots_of(k, table, b, n)
            qq = q[b].double().unflatten(0, (hk, group))
            s = torch.einsum("hgtd,hnd->hgtn", qq, kk) * sc
            ll = lse[b].double().unflatten(0, (hk, group))[..., None]
            p = torch.where(ll == -math.inf, 0.0, torch.exp(s - ll))
            size = torch.einsum("hgtd,hnd->hgtn", qq.abs(), kk.abs()) * sc + ll.abs().nan_to_num(posinf=0)
            err = (p * (score_error(size, dim) + (group * t + 8) * LN)).sum((1, 2))
            want = before[b, :, :n].double() + p.sum((1, 2))
            assert ((weights[b, :, :n].double() - want).abs() <= err + 2 * LN * want).all()
            assert torch.equal(weights[b, :, n:], before[b, :, n:])
    assert read_status() == 0


@gpu
def test_weights_of_a_row_add_up():
    """What the queries give the cache and keep for the tree is all that there is."""
    g = torch.Generator().manual_seed(16)
    lengths = [100, 250]
    k, v, table, ns = make_cache(lengths, 2, 64, 16, F16)
    q = torch.randn(2, 4, 6, 64, generator=g).half().cuda()
    kt, vt = (torch.randn(2, 2, 6, 64, generator=g).half().cuda() for _ in range(2))
    _, lse = fa.tree_attention(q, k, v, table, ns, kt, vt)
    weights = torch.zeros(2, 2, table.shape[1] * 16).cuda()
    fa.accumulate_attention_weight(weights, q, k, table, ns, lse)
    _, alone = fa.tree_attention(q, k, v, table, ns)
    share = torch.exp(alone.double() - lse.double()).unflatten(1, (2, 2)).sum((2, 3))
    torch.testing.assert_close(weights.double().sum(-1), share, rtol=1e-5, atol=0)


# ------------------------------------------------------------------ evict (GPU)

def evict_64(w, pos, n, budget, recent, sinks):
    """Where each slot of the smaller cache comes from."""
    if n <= budget:
        return list(range(n))
    last = max(pos[:n])
    rank = []
    for i in range(n):
        safe = pos[i] > last - recent or pos[i] < sinks
        value = math.inf if safe else -math.inf if math.isnan(w[i]) else w[i]
        # protected before anything, NaN behind anything
        rank.append(((0 if safe else 2 if math.isnan(w[i]) else 1), -value, i))
    kept = sorted(x[2] for x in sorted(rank)[:budget])
    src = list(range(budget))
    inside = set(kept)
    holes = [i for i in range(budget) if i not in inside]
    for to, come in zip(holes, [i for i in kept if i >= budget]):
        src[to] = come
    return src


EVICTS = [  # lengths, kv heads, budget, recent, sinks, page, dim
    ([1], 1, 1, 0, 0, 16, 64),
    ([2], 1, 1, 1, 0, 16, 64),
    ([0, 5, 16, 17, 40], 2, 16, 4, 2, 16, 64),
    ([33, 90], 3, 32, 0, 0, 32, 128),
    ([64, 65, 200], 1, 64, 64, 0, 16, 64),   # only the last positions stay
    ([64, 65, 200], 1, 64, 0, 64, 16, 64),   # only the first
    ([1500, 1029], 2, 1024, 100, 4, 48, 64),
    ([5000], 1, 700, 50, 4, 16, 64),
    ([300], 2, 5000, 0, 0, 16, 64),          # a budget above the slots
]


def check_evict(lengths, hk, budget, recent, sinks, page, dim, weights, positions, dtype=F16):
    k, v, table, ns = make_cache(lengths, hk, dim, page, dtype)
    k0, v0, w0, p0 = k.clone(), v.clone(), weights.clone(), positions.clone()
    w, p, n_new = fa.evict_from_cache(k, v, table, ns, weights, positions, budget, recent=recent,
                                      sinks=sinks)
    assert torch.equal(weights.nan_to_num(-7), w0.nan_to_num(-7)) and torch.equal(positions, p0)
    assert ns.tolist() == list(lengths) and n_new.tolist() == [min(n, budget) for n in lengths]
    untouched = torch.ones(k.shape[:3], dtype=torch.bool)
    wl, pl = weights.tolist(), positions.tolist()
    for b, n in enumerate(lengths):
        for h in range(hk):
            src = evict_64(wl[b][h], pl[b][h], n, budget, recent, sinks)
            m = len(src)
            assert torch.equal(w[b, h, :m].nan_to_num(-7), weights[b, h, src].nan_to_num(-7))
            assert torch.equal(p[b, h, :m], positions[b, h, src])
            assert (w[b, h, m:] == 0).all() and (p[b, h, m:] == -1).all()
            for x, x0 in ((k, k0), (v, v0)):
                assert torch.equal(slots_of(x, table, b, m)[h], slots_of(x0, table, b, n)[h, src])
            for s in range(m):
                untouched[int(table[b, s // page]), h, s % page] = False
    for x, x0 in ((k, k0), (v, v0)):  # what lies behind the new length and in other pages
        assert torch.equal(x[untouched].view(torch.int16), x0[untouched].view(torch.int16))
    assert read_status() == 0


def _slots(lengths, hk, page, seed):
    g = torch.Generator().manual_seed(seed)
    slots = max(1, -(-max(lengths) // page)) * page
    weights = torch.rand(len(lengths), hk, slots, generator=g)
    positions = torch.stack([torch.stack([torch.cat([torch.randperm(n, generator=g),
                                                     torch.full((slots - n,), 1 << 30)])
                                          for _ in range(hk)]) for n in lengths]).int()
    return weights, positions


@gpu
@pytest.mark.parametrize("case", EVICTS)
def test_evict(case):
    lengths, hk, *_, page, dim = case
    weights, positions = _slots(lengths, hk, page, 17)
    check_evict(*case, weights.cuda(), positions.cuda(), BF16 if dim == 128 else F16)


@gpu
@pytest.mark.parametrize("kind", ["equal", "zeros", "few values", "odd numbers", "one bit apart"])
def test_evict_ties_and_odd_weights(kind):
    case = ([900, 40, 513], 2, 200, 10, 3, 16, 64)
    weights, positions = _slots(case[0], 2, 16, 18)
    g = torch.Generator().manual_seed(19)
    if kind == "equal":
        weights.fill_(0.5)
    elif kind == "zeros":  # both zeros are one value
        weights = torch.where(torch.rand(weights.shape, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "few values":
        weights = (weights * 3).floor()
    elif kind == "one bit apart":
        weights = (torch.randint(0, 40, weights.shape, generator=g) + 0x3F800000).int().view(torch.float32)
    else:
        for value, share in ((math.nan, 0.3), (math.inf, 0.02), (-math.inf, 0.2), (-3.0, 0.1), (1e-42, 0.1)):
            weights = torch.where(torch.rand(weights.shape, generator=g) < share, value, weights)
    check_evict(*case, weights.cuda(), positions.cuda())


@gpu
def test_evict_long_sequence_over_a_cluster():
    """Enough slots for eight blocks to share one selection, kept in shared memory, and so many
    that they are not."""
    for n, budget in ((40000, 9000), (500000, 200000)):
        g = torch.Generator(device="cuda").manual_seed(20)
        k = torch.arange(n, device="cuda").half().reshape(1, 1, n, 1).expand(1, 1, n, 64).contiguous()
        v = k.neg()
        k0 = k.clone()
        weights = torch.rand(1, 1, n, generator=g, device="cuda")
        positions = torch.randperm(n, generator=g, device="cuda").int().reshape(1, 1, n)
        table, ns = torch.zeros(1, 1).int().cuda(), torch.tensor([n]).int().cuda()
        w, p, m = fa.evict_from_cache(k, v, table, ns, weights, positions, budget, recent=1000, sinks=10)
        src = torch.tensor(evict_64(weights[0, 0].tolist(), positions[0, 0].tolist(), n, budget, 1000, 10))
        src = src.cuda()
        assert m.tolist() == [budget]
        assert torch.equal(w[0, 0, :budget], weights[0, 0, src])
        assert torch.equal(p[0, 0, :budget], positions[0, 0, src])
        assert torch.equal(k[0, 0, :budget], k0[0, 0, src]) and torch.equal(k[0, 0, budget:], k0[0, 0, budget:])
        assert torch.equal(v, k.neg())


@gpu
@pytest.mark.parametrize("n, hk, budget, page, dim", [
    (40000, 1, 9000, 40000, 64), (500000, 1, 200000, 16, 64), (70000, 3, 30000, 112, 128),
    (9000, 40, 5000, 48, 64), (3000, 70, 1500, 16, 128), (30000, 160, 29000, 64, 64)])
def test_evicted_rows_come_from_their_slots(n, hk, budget, page, dim):
    """Selections by eight, four, two and one blocks, of slots in shared memory and of too many for
    it: a row's elements spell its slot and head."""
    g = torch.Generator().manual_seed(23)
    per = -(-n // page)
    at = torch.arange(per * page, device="cuda")
    digits = [at % 1000, at // 1000]  # each exact in fp16
    table = torch.randperm(per + 2, generator=g)[None, :per].int().cuda()
    k = torch.zeros(per + 2, hk, page, dim, dtype=F16, device="cuda")
    for i, x in enumerate(digits):
        k[table[0].long(), :, :, i::3] = x.half().reshape(per, 1, page, 1)
    k[:, :, :, 2::3] = torch.arange(hk, device="cuda").half()[:, None, None]
    v = k.flip(-1).neg()
    k0 = k.clone()
    weights = torch.rand(1, hk, per * page, generator=g)
    positions = torch.stack([torch.randperm(per * page, generator=g) for _ in range(hk)])[None].int()
    ns = torch.tensor([n], dtype=torch.int32).cuda()
    w, p, m = fa.evict_from_cache(k, v, table, ns, weights.cuda(), positions.cuda(), budget, recent=100, sinks=5)
    assert m.tolist() == [budget] and read_status() == 0

    def rows(pages):  # [H_kv, slots, D]
        return pages[table[0].long()].transpose(0, 1).flatten(1, 2)

    for h in range(0, hk, max(1, hk // 3)):
        src = torch.tensor(evict_64(weights[0, h].tolist(), positions[0, h].tolist(), n, budget, 100, 5))
        assert (src >= budget).any()
        assert torch.equal(w[0, h, :budget].cpu(), weights[0, h, src])
        assert torch.equal(p[0, h, :budget].cpu(), positions[0, h, src])
        assert torch.equal(rows(k)[h, :budget], rows(k0)[h, src.cuda()])
        assert torch.equal(rows(k)[h, budget:], rows(k0)[h, budget:])
    assert torch.equal(v, k.flip(-1).neg())


# ------------------------------------------------------------------ device-side checks (GPU)

@gpu
@ROOM
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("t", [3, 40, 150])
def test_bad_pages_of_many_rows(t, dim, room):
    """A page that does not exist in the middle of a tile of keys, for every kernel."""
    read_status()
    lengths = [300, 40]
    k, v, table, ns = make_cache(lengths, 1, dim, 32, F16)
    table = table_of(table, room, 32, 2 * t)
    q = torch.randn(2, 1, t, dim, generator=torch.Generator().manual_seed(22)).half().cuda()
    table[0, 5] = k.shape[0]
    out, lse = fa.tree_attention(q, k, v, table, ns)
    assert read_status() == CACHE_BIT
    table[0, 5] = 0
    keep = torch.tensor([s for s in range(300) if not 160 <= s < 192])
    kk, vv = slots_of(k, table, 0, 300)[:, keep].cpu(), slots_of(v, table, 0, 300)[:, keep].cpu()
    ref = attention_64(q[0].cpu(), kk, vv, torch.ones(t, len(keep), dtype=torch.bool), dim ** -0.5)
    check_attention((out[:1], lse[:1]), [x[None] for x in ref], F16, dim)


@gpu
def test_bad_tables_and_lengths_are_left_out_and_reported():
    """The status bit is set, the rows of a bad page are left out, nothing else changes."""
    read_status()
    lengths = [60, 40]
    k, v, table, ns = make_cache(lengths, 1, 64, 16, F16)
    q = torch.randn(2, 1, 1, 64, generator=torch.Generator().manual_seed(21)).half().cuda()
    for entry in (-1, k.shape[0], 1 << 30):
        bad = table.clone()
        bad[0, 1] = entry
        out, lse = fa.tree_attention(q, k, v, bad, ns)
        assert read_status() == CACHE_BIT
        keep = torch.tensor([s for s in range(60) if not 16 <= s < 32])
        kk, vv = slots_of(k, table, 0, 60)[:, keep].cpu(), slots_of(v, table, 0, 60)[:, keep].cpu()
        ref = attention_64(q[0].cpu(), kk, vv, torch.ones(1, 44, dtype=torch.bool), 0.125)
        check_attention((out[:1], lse[:1]), [x[None] for x in ref], F16, 64)
        weights = torch.zeros(2, 1, table.shape[1] * 16).cuda()
        fa.accumulate_attention_weight(weights, q, k, bad, ns, lse)
        assert read_status() == CACHE_BIT and (weights[0, 0, 16:32] == 0).all()
        k1, v1 = k.clone(), v.clone()
        key = torch.ones(2, 1, 3, 64, dtype=F16).cuda()
        new = fa.append_to_cache(key, key, k1, v1, bad, torch.tensor([15, 40]).int().cuda())
        assert read_status() == CACHE_BIT and new.tolist() == [18, 43]
        assert (k1[int(table[0, 0]), 0, 15] == 1).all()
    for length in (-3, table.shape[1] * 16 + 1):
        wrong = torch.tensor([length, 40]).int().cuda()
        out, lse = fa.tree_attention(q, k.nan_to_num(), v.nan_to_num(posinf=1.0), table, wrong)
        assert read_status() == CACHE_BIT and out.isfinite().all()
    for counts, path in (([4, 0], None), ([-1, 0], None), ([2, 0], [[7, 0, 0], [0, 0, 0]])):
        k1, v1 = k.clone(), v.clone()
        fa.append_to_cache(key, key, k1, v1, table, ns * 0, counts=torch.tensor(counts).int().cuda(),
                           path=None if path is None else torch.tensor(path).int().cuda())
        assert read_status() == CACHE_BIT
    full = torch.tensor([table.shape[1] * 16 - 1, 0]).int().cuda()
    new = fa.append_to_cache(key, key, k.clone(), v.clone(), table, full)
    assert read_status() == CACHE_BIT and new.tolist() == [table.shape[1] * 16, 3]
    wrong = torch.tensor([60, 40]).int().cuda()
    sizes = torch.tensor([2, 1]).int().cuda()
    fa.tree_attention(q, k, v, table, wrong, key[:, :, :1], key[:, :, :1], tree_sizes=sizes)
    assert read_status() == CACHE_BIT


@gpu
@ROOM
def test_offsets_past_32_bits(room):
    """The same cache at the end of pages of more than 2^32 elements: the same bits."""
    lengths = [700, 33, 1500]
    g = torch.Generator().manual_seed(29)
    k, v, table, ns = make_cache(lengths, 2, 128, 64, F16, room=70)
    pages = (1 << 32) // (2 * 64 * 128) + k.shape[0] + 1
    far_k, far_v = (torch.empty(pages, 2, 64, 128, dtype=F16, device="cuda") for _ in range(2))
    behind = pages - k.shape[0]
    far_k[behind:], far_v[behind:] = k, v
    slots = table.shape[1] * 64
    weights = torch.rand(3, 2, slots, generator=g).cuda()
    positions = torch.arange(slots, dtype=torch.int32).repeat(3, 2, 1).cuda()
    q, kt, vt = (torch.randn(3, h, 65, 128, generator=g).half().cuda() for h in (8, 2, 2))
    new = torch.arange(65, dtype=torch.int32).repeat(3, 1).cuda()

    def step(k, v, table):
        w, at = weights.clone(), positions.clone()
        out, lse = fa.tree_attention(q, k, v, table_of(table, room, 64, 3 * 8 * 65), ns, kt, vt)
        fa.accumulate_attention_weight(w, q, k, table, ns, lse)
        longer = fa.append_to_cache(kt, vt, k, v, table, ns, None, None, w, at, new)
        rest = fa.evict_from_cache(k, v, table, longer, w, at, 300, 10, 2)
        again = fa.tree_attention(q[:, :, :1], k, v, table, rest[2])
        return [out, lse, longer, *rest, *again]

    for a, b in zip(step(far_k, far_v, table + behind), step(k, v, table)):
        assert torch.equal(a, b)
    assert torch.equal(far_k[behind:].view(torch.int16), k.view(torch.int16))
    assert torch.equal(far_v[behind:].view(torch.int16), v.view(torch.int16))


@gpu
def test_a_cache_without_slots():
    k, v, table, ns = make_cache([0, 0], 2, 64, 16, F16)
    none = table[:, :0]
    weights = torch.zeros(2, 2, 0).cuda()
    positions = torch.zeros(2, 2, 0, dtype=torch.int32).cuda()
    w, at, rest = fa.evict_from_cache(k, v, none, ns, weights, positions, 3)
    assert w.shape == at.shape == (2, 2, 0) and rest.tolist() == [0, 0]
    rows = torch.zeros(2, 2, 0, 64, dtype=F16).cuda()
    assert fa.append_to_cache(rows, rows, k, v, none, ns).tolist() == [0, 0]
    q = torch.zeros(2, 2, 1, 64, dtype=F16).cuda()
    assert fa.accumulate_attention_weight(weights, q, k, none, ns, torch.zeros(2, 2, 1).cuda()) is not None


@gpu
def test_append_of_one_row_twice():
    k, v, table, ns = make_cache([5], 1, 64, 16, F16, room=8)
    rows = torch.randn(1, 1, 3, 64, generator=torch.Generator().manual_seed(31)).half().cuda()
    path = torch.tensor([[2, 2, 0]], dtype=torch.int32).cuda()
    assert fa.append_to_cache(rows, -rows, k, v, table, ns, path).tolist() == [8]
    for pages, x in ((k, rows), (v, -rows)):
        got = torch.stack([pages[int(table[0, s // 16]), 0, s % 16] for s in (5, 6, 7)])
        assert torch.equal(got, x[0, 0, [2, 2, 0]])
