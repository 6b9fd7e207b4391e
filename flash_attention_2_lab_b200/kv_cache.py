"""Serving from a paged key/value cache on the sm_100a kernels.

A cache is plain tensors that the caller holds:

* ``k_pages``, ``v_pages``: [pages, H_kv, page_size, D], float16 or bfloat16, D 64 or 128,
  page_size a multiple of 16;
* ``block_table``: int32 [B, pages of a sequence], ``lengths``: int32 [B].  Slot ``s`` of
  sequence ``b`` is row ``s % page_size`` of page ``block_table[b, s // page_size]``,
  ``s < lengths[b]``.  One contiguous [B, H_kv, capacity, D] tensor is a cache with page_size =
  capacity and the table ``arange(B)[:, None]``;
* for eviction ``weights`` (float32) and ``positions`` (int32), [B, H_kv, slots of a sequence].

A decoding step turns queries and keys by their positions (``rotary.apply_rotary``), attends
with ``tree_attention`` over the cache and the step's own keys, and appends the keys that stay:
all of them, or the accepted path of a drafted tree (``append_to_cache``).  Where the cache is to
keep its size, ``accumulate_attention_weight`` follows each attention and ``evict_from_cache``
runs when the cache has grown past its budget.

Lengths stay on the device: no call waits for it.  The kernels check every length and table
entry that they use; one that leads outside the cache is not followed, the rows that it stands
for are left out, and bit 32 of the device status word (``lib().fa_read_status``) is set.
``check_cache`` does the same check on the host.  Calls that change a cache need a page to stand
once in the table; ``tree_attention`` and ``accumulate_attention_weight`` may read shared ones.

Nothing here is differentiable, and the reference has no counterpart (it has no cache).
"""

from __future__ import annotations

import torch

from ._native import ext


def tree_attention(query, k_pages, v_pages, block_table, lengths, k_tree=None, v_tree=None,
                   tree_mask=None, tree_sizes=None, scale: float | None = None):
    """(out, lse) of queries [B, H, T, D] over the cache and the tree's own keys.

    Query ``t`` of head ``h`` sees the cached slots of kv head ``h // (H / H_kv)`` and the rows
    ``j`` of ``k_tree``, ``v_tree`` [B, H_kv, T, D] where ``tree_mask`` (bool [T, T] or
    [B, T, T]) is true at ``[t, j]``; without a mask ``j <= t``, a chain, which is also how a
    chunk of a prompt is attended.  One token and no tree is plain decoding over the cache.
    ``tree_sizes`` (int32 [B]): of sequence ``b`` only the first ``tree_sizes[b]`` tokens are
    there.  A token that is not there or sees nothing gets 0, its lse -inf.

    out has the dtype of query; lse is float32 [B, H, T], natural log.  The scale is positive,
    by default 1/sqrt(D).  Scores and sums are in 32 bits; the probabilities are rounded to the
    dtype of v_pages for their product with the values, which adds up to half a step of it
    (relative) to each, and the output is rounded once.

    Query and tree tensors may have any strides; where their rows cannot be loaded 16 bytes at a
    time they are copied first.  A long chunk pays for all T x T pairs of its own tokens, hidden
    ones too: attend one of thousands of tokens over a short cache in pieces.  The kernel is
    chosen by the slots that the table has room for, as the lengths stay on the device.
    """
    return tuple(ext().tree_attention(query, k_pages, v_pages, block_table, lengths, k_tree, v_tree,
                                      tree_mask, tree_sizes, scale))


def append_to_cache(key, value, k_pages, v_pages, block_table, lengths, path=None, counts=None,
                    weights=None, positions=None, new_positions=None):
    """Writes rows of key and value [B, H_kv, N, D] behind each sequence's slots and returns the
    new lengths (``lengths`` itself is not changed).

    Row ``path[b, i]`` (int32 [B, N]; None: row ``i``) becomes slot ``lengths[b] + i`` for
    ``i < counts[b]`` (int32 [B]; None: N): the accepted nodes of a drafted tree, in order.  The
    rows end before the first entry of the path that names none of the N, and where the table
    has no more slots; the new lengths say how many were taken.
    ``weights`` get 0 at the new slots and ``positions`` get ``new_positions[b, path[b, i]]``
    (int32 [B, N]), if given.
    """
    return ext().append_to_cache(key, value, k_pages, v_pages, block_table, lengths, path, counts,
                                 weights, positions, new_positions)


def accumulate_attention_weight(weights, query, k_pages, block_table, lengths, lse,
                                scale: float | None = None):
    """Adds to ``weights``, in place, what each cached slot weighed in an attention of ``query``
    [B, H, T, D] that returned ``lse``: the sum of ``exp(scale q . k - lse)`` over the heads of
    the kv head and the tokens.  Queries with an lse of -inf add nothing.  Returns ``weights``.
    """
    return ext().accumulate_attention_weight(weights, query, k_pages, block_table, lengths, lse, scale)


def evict_from_cache(k_pages, v_pages, block_table, lengths, weights, positions, budget: int,
                     recent: int = 0, sinks: int = 0):
    """Cuts every (sequence, kv head) to ``budget`` slots; returns its new (weights, positions,
    lengths), while the pages change in place.

    What stays: positions below ``sinks``, the ``recent`` last positions (above the largest
    position minus ``recent``), then the largest weights; the lowest slot of equal ones, NaN last
    of all.  Kept slots behind the budget move into dropped ones before it, in slot order; the
    others keep their place, so slots are in no order afterwards - attention does not ask for
    one - and ``positions`` says where each came from.  Behind the new length weights are 0 and
    positions -1.  A move from or into a slot whose page does not exist is left out, weight and
    position with it.
    """
    return tuple(ext().evict_from_cache(k_pages, v_pages, block_table, lengths, weights, positions,
                                        budget, recent, sinks))


def tree_mask_from_parents(parents):
    """The mask of trees given by their parents (integers [..., T], a negative number for a root,
    and below ``t`` for node ``t``): bool [..., T, T], true where ``j`` is ``t`` or above it."""
    if parents.dim() < 1:
        raise ValueError("parents must have shape [..., T]")
    n = parents.shape[-1]
    at = torch.arange(n, device=parents.device)
    if bool((parents >= at).any()):
        raise ValueError("a node's parent must come before it")
    # self or parent; squaring doubles the generations that a node sees
    mask = (at[:, None] == at) | (parents[..., None] == at)
    for _ in range(max(n - 1, 1).bit_length()):
        mask = (mask.float() @ mask.float()) > 0
    return mask


def check_cache(k_pages, block_table, lengths) -> None:
    """Raises ValueError for lengths that the table cannot address and for entries, among those
    that the lengths use, that name no page.  Reads them on the host, so it waits for the device.
    """
    pages, page_size = k_pages.shape[0], k_pages.shape[2]
    n, table = lengths.cpu().long(), block_table.cpu().long()
    slots = table.shape[1] * page_size
    bad = ((n < 0) | (n > slots)).nonzero().flatten()
    if len(bad):
        b = int(bad[0])
        raise ValueError(f"length {int(n[b])} of sequence {b} is not in [0, {slots}]")
    used = torch.arange(table.shape[1]) * page_size < n[:, None]
    bad = (used & ((table < 0) | (table >= pages))).nonzero()
    if len(bad):
        b, i = bad[0].tolist()
        raise ValueError(f"page {int(table[b, i])} of sequence {b}, entry {i}, is not in [0, {pages})")
