"""A key-value cache in pages for several requests at once, and attention over it.

The reference keeps one contiguous cache per request (HuggingFace's, `adapters/huggingface.py:106-202`) and has no counterpart of
this. Here the keys and values of a layer are `(n_pages, page_size, kv_heads, head_dim)` tensors that all requests share, and a block
table says which pages hold a request. One serving step is

    step = assign_pages(new_lens, lens, ...)        # once: pages for the new tokens, their slots and positions
    store_paged(keys, values, ..., step.slot_map)   # every layer
    paged_attention(queries, ..., step.kv_lens, step.cu_new, ...)

on tokens packed request after request, chunks of prompts and single tokens side by side. Nothing reads the device back, so a step
can be captured into a graph. `PagedKVCache` keeps the tensors together. The kernels run on the current stream of the
tensors' device; there is no gradient.

A cache may be held in 8 bits: `torch.float8_e4m3fn` tensors of the same shape and, for keys and for values, `torch.float8_e8m0fnu` scales
`(n_pages, kv_heads, page_size)`, powers of two (`include/sah_pages.h` has the rule). Where a function takes `key_scales` and `value_scales`, they go
with such a cache. `load_paged` reads contexts back, as the contiguous tensors that the maskers and `ResearchAttention` take.

A token may attend to a few pages instead of all: `update_page_bounds` keeps the smallest and largest element of every channel of the pages'
keys, `select_pages` chooses a token's pages by how large a logit they can hold (the score of Quest, Tang et al., 2024, which the reference has as a masker:
`maskers/fixed/implementations/quest_top_k.py:58`), `paged_attention(..., pages=...)` attends to them.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from ... import _native as N


class PageAssignment(NamedTuple):
    """Where a step's new tokens go. Device tensors; `include/sah_serve.h` has the rules."""

    slot_map: torch.Tensor    # int64 [n_tokens]: page * page_size + entry, or -1
    positions: torch.Tensor   # int32 [n_tokens]: the token's position in its request
    cu_new: torch.Tensor      # int32 [n_requests + 1]: request b's rows are cu_new[b] .. cu_new[b + 1] - 1
    kv_lens: torch.Tensor     # int32 [n_requests]: tokens a request holds after the step; 0 where it was not granted
    granted: torch.Tensor     # bool [n_requests]


def _check(t: torch.Tensor, what: str, dtype: torch.dtype, size: Optional[int], device: torch.device) -> None:
    """A contiguous tensor of one dimension, of this type and size (None: any) on this device."""
    if isinstance(t, torch.Tensor) and t.dtype == dtype and t.dim() == 1 and t.device == device and t.is_contiguous() \
            and (size is None or t.shape[0] == size):
        return  # (one line for the call that is as it should be: a step makes a dozen of them)
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if t.dim() != 1 or size is not None and t.shape[0] != size:
        raise ValueError(f"{what} must have shape ({'n' if size is None else size},), got {tuple(t.shape)}")
    raise ValueError(f"{what} must be contiguous")


def _check_table(block_table: torch.Tensor, n_requests: int, device: torch.device) -> None:
    if block_table.device != device or block_table.dtype != torch.int32:
        raise ValueError(f"block_table must be int32 on {device}, got {block_table.dtype} on {block_table.device}")
    if block_table.dim() != 2 or block_table.shape[0] != n_requests or block_table.shape[1] == 0:
        raise ValueError(f"block_table must have shape ({n_requests}, pages), got {tuple(block_table.shape)}")
    if (block_table.stride(1) != 1 and block_table.shape[1] > 1) or (n_requests > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError("block_table's rows must be contiguous and apart")


def _check_page_size(page_size: int) -> None:
    if not 1 <= page_size < 2 ** 31:  # (a wider number would lose its upper half on the way to the kernels)
        raise ValueError(f"page_size must be in [1, 2^31), got {page_size}")


_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _check_scales(scales: Optional[torch.Tensor], what: str, cache: torch.Tensor) -> None:
    """Scales where the cache is in 8 bits, none where it is not."""
    if cache.dtype != _E4M3:
        if scales is not None:
            raise ValueError(f"{what} go with a {_E4M3} cache, this one is {cache.dtype}")
        return
    pages, page_size, heads, _ = cache.shape
    if isinstance(scales, torch.Tensor) and scales.dtype == _E8M0 and scales.shape == (pages, heads, page_size) and scales.device == cache.device \
            and scales.is_contiguous():
        return
    got = f"{scales.dtype} {tuple(scales.shape)} on {scales.device}" if isinstance(scales, torch.Tensor) else type(scales).__name__
    raise ValueError(f"{what} of a {_E4M3} cache must be contiguous {_E8M0} ({pages}, {heads}, {page_size}) on {cache.device}, got {got}")


def _cache_block(key_cache: torch.Tensor, value_cache: Optional[torch.Tensor], key_scales: Optional[torch.Tensor],
                 value_scales: Optional[torch.Tensor]) -> N.PageCache:
    dtype = N.SAH_E4M3 if key_cache.dtype == _E4M3 else N.dtype_code(key_cache.dtype)
    pages, page_size, heads, dim = key_cache.shape
    v = key_cache if value_cache is None else value_cache
    return N.PageCache(key_cache.data_ptr(), *key_cache.stride()[:3], v.data_ptr(), *v.stride()[:3], N.ptr(key_scales),
                       N.ptr(key_scales if value_cache is None else value_scales), dtype, pages, page_size, heads, dim)


def _pitch(block_table: torch.Tensor) -> int:
    return max(block_table.stride(0), block_table.shape[1])  # one row: its stride says nothing


def _check_cache(key_cache: torch.Tensor, value_cache: torch.Tensor) -> None:
    N.require_device(key_cache, "key_cache")
    if key_cache.dim() != 4 or key_cache.shape != value_cache.shape:
        raise ValueError("key_cache and value_cache must both be (n_pages, page_size, kv_heads, head_dim), got "
                         f"{tuple(key_cache.shape)} and {tuple(value_cache.shape)}")
    if value_cache.device != key_cache.device or value_cache.dtype != key_cache.dtype:
        raise ValueError("key_cache and value_cache must be of one type on one device")
    if key_cache.shape[3] > 1 and (key_cache.stride(3) != 1 or value_cache.stride(3) != 1):
        raise ValueError("the caches' innermost stride must be 1")


def assign_pages(new_lens: torch.Tensor, lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 free_count: torch.Tensor, page_size: int, n_tokens: int, lens_out: Optional[torch.Tensor] = None,
                 free_count_out: Optional[torch.Tensor] = None) -> PageAssignment:
    """Pages, slots and positions for the `new_lens[b]` tokens that each request gets in this step.

    A request that holds `lens[b]` tokens needs pages where those end; they come off the end of
    `free_pages[:free_count]`, request after request, and are entered into `block_table`. A request is granted all its tokens or none
    (`granted`): where they do not fit into the table's width or into `n_tokens` rows, or, among requests that need pages, from
    the first on for which there are too few. `n_tokens` is the number of token rows the program has packed (more than the requests' sum is a
    padded batch: slot -1, position 0). `lens` and `free_count` are brought up to date in place unless `lens_out` /
    `free_count_out` are given. int32 tensors; at most 4096 requests.
    """
    N.require_device(new_lens, "new_lens")
    device, n = new_lens.device, new_lens.shape[0] if new_lens.dim() == 1 else -1
    lens_out = lens if lens_out is None else lens_out
    free_count_out = free_count if free_count_out is None else free_count_out
    _check(new_lens, "new_lens", torch.int32, None, device)
    if n == 0:
        raise ValueError("assign_pages needs at least one request")
    _check(lens, "lens", torch.int32, n, device)
    _check(lens_out, "lens_out", torch.int32, n, device)
    _check(free_pages, "free_pages", torch.int32, None, device)
    _check(free_count, "free_count", torch.int32, 1, device)
    _check(free_count_out, "free_count_out", torch.int32, 1, device)
    _check_table(block_table, n, device)
    _check_page_size(page_size)
    if not 0 <= n_tokens <= 2 ** 30:
        raise ValueError(f"n_tokens must be in [0, 2^30], got {n_tokens}")
    slot_map = torch.empty(n_tokens, dtype=torch.int64, device=device)
    # one allocation for the int32 outputs and the kernels' records
    words = torch.empty(n_tokens + 4 * n + 1, dtype=torch.int32, device=device)
    work, cu_new, kv_lens, positions = words.split_with_sizes((2 * n, n + 1, n, n_tokens))
    granted = torch.empty(n, dtype=torch.bool, device=device)
    N.call_on(device, "sah_paged_assign", N.PagedAssignArgs(
        new_lens.data_ptr(), lens.data_ptr(), block_table.data_ptr(), _pitch(block_table), block_table.shape[1],
        free_pages.data_ptr(), free_count.data_ptr(), free_pages.shape[0], n, page_size, n_tokens,
        slot_map.data_ptr(), positions.data_ptr(), cu_new.data_ptr(), kv_lens.data_ptr(), granted.data_ptr(),
        lens_out.data_ptr(), free_count_out.data_ptr(), work.data_ptr(), N.stream_ptr(device)))
    return PageAssignment(slot_map, positions, cu_new, kv_lens, granted)


def release_pages(finished: torch.Tensor, lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, page_size: int) -> None:
    """Gives the pages of every request with `finished[b]` (bool) back to `free_pages`: its length becomes 0, its table entries -1,
    and its row can serve another request. Entries that are negative already (no page) are not given back."""
    N.require_device(finished, "finished")
    device, n = finished.device, finished.shape[0] if finished.dim() == 1 else -1
    _check(finished, "finished", torch.bool, None, device)
    if n == 0:
        raise ValueError("release_pages needs at least one request")
    _check(lens, "lens", torch.int32, n, device)
    _check(free_pages, "free_pages", torch.int32, None, device)
    _check(free_count, "free_count", torch.int32, 1, device)
    _check_table(block_table, n, device)
    _check_page_size(page_size)
    work = torch.empty(2 * n, dtype=torch.int32, device=device)
    N.call_on(device, "sah_paged_release", N.PagedReleaseArgs(
        finished.data_ptr(), lens.data_ptr(), block_table.data_ptr(), _pitch(block_table), block_table.shape[1],
        free_pages.data_ptr(), free_count.data_ptr(), free_pages.shape[0], n, page_size, work.data_ptr(), N.stream_ptr(device)))


def store_paged(keys: torch.Tensor, values: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                slot_map: torch.Tensor, *, key_scales: Optional[torch.Tensor] = None, value_scales: Optional[torch.Tensor] = None) -> None:
    """Writes `keys[t]` and `values[t]`, `(n_tokens, kv_heads, head_dim)`, to slot `slot_map[t]` of the caches; rows with a slot of -1
    (or any other outside the cache) are passed over. No two rows may name the same slot: which of them it would hold is
    not defined. An 8-bit cache takes float32, bfloat16 or float16 rows (addresses and strides multiples of 16 bytes, head_dim of
    16): each is rounded once to e4m3 times the least power of two, from 2^-110 up, at which its largest element fits; what is not finite
    becomes NaN, and magnitudes from 248 * 2^120 (3.297e38) on are rounded to 2^128: infinite when they are read."""
    _check_cache(key_cache, value_cache)
    _check_scales(key_scales, "key_scales", key_cache)
    _check_scales(value_scales, "value_scales", value_cache)
    device = key_cache.device
    pages, page_size, heads, dim = key_cache.shape
    narrow = key_cache.dtype == _E4M3
    rows, dtype = (keys.shape[0] if keys.dim() else 0, heads, dim), keys.dtype if narrow else key_cache.dtype
    for t, what in ((keys, "keys"), (values, "values")):
        if t.device != device or t.dtype != dtype:
            raise ValueError(f"{what} must be {dtype} on {device}, got {t.dtype} on {t.device}")
        if t.shape != rows:
            raise ValueError(f"{what} must have shape (n_tokens, {heads}, {dim}), got {tuple(t.shape)}")
        if t.stride(2) != 1 and dim > 1:
            raise ValueError(f"{what}: the innermost stride must be 1")
    _check(slot_map, "slot_map", torch.int64, rows[0], device)
    if narrow:
        N.call_on(device, "sah_page_store", N.PageStoreArgs(
            _cache_block(key_cache, value_cache, key_scales, value_scales), keys.data_ptr(), keys.stride(0), keys.stride(1),
            values.data_ptr(), values.stride(0), values.stride(1), slot_map.data_ptr(), N.dtype_code(dtype), rows[0], N.stream_ptr(device)))
        return
    N.call_on(device, "sah_paged_store", N.PagedStoreArgs(
        keys.data_ptr(), keys.stride(0), keys.stride(1), values.data_ptr(), values.stride(0), values.stride(1),
        key_cache.data_ptr(), *key_cache.stride()[:3], value_cache.data_ptr(), *value_cache.stride()[:3],
        slot_map.data_ptr(), N.dtype_code(dtype), rows[0], heads, dim, pages, page_size, N.stream_ptr(device)))


def paged_attention(queries: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, cu_new: torch.Tensor, scaling: float, *, max_context: Optional[int] = None,
                    sink_size: int = 0, window_size: int = 0, sinks: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, pages: Optional[torch.Tensor] = None,
                    key_scales: Optional[torch.Tensor] = None, value_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of packed new tokens `(n_tokens, heads, head_dim)` over the cache, which holds their keys already.

    Row `cu_new[b] + i` stands at position `kv_lens[b] - new_b + i` of request b, `new_b = cu_new[b + 1] - cu_new[b]`, and sees the request's
    keys up to its own; with `window_size > 0` of those only the first `sink_size` and the last `window_size`, the columns of
    `SinkMasker` and `LocalMasker`. `sinks` (float32 `(heads,)`): a logit per head in the denominator. Query heads share key heads in
    groups, as `repeat_kv` would have it. A row that sees nothing is 0; rows behind the last request's keep what `out` held (without
    `out`: unspecified). `max_context`, about the longest request's length, decides how work is split (default: the
    table's width); results do not depend on it beyond the order of sums. head_dim a multiple of 8 up to 256, page_size a power of two,
    addresses and strides multiples of 16 bytes; `out` shares no memory with the other tensors (refused; it and
    the queries may be slices of one buffer, their tokens equally far apart). Returns `(n_tokens, heads, head_dim)`.

    An 8-bit cache (head_dim a multiple of 16) takes float32, bfloat16 or float16 queries, the result's type. Long chunks under 16-bit ones are attended
    to through a copy of their contexts, from 256 MiB on with room for `max_context` tokens of every request, 2 GiB at most: where the table is much wider, what
    the step's longest request has saves memory (a longer context costs time, and changes nothing else than whether weights are rounded to 16 bits). `pages`, int32 `(n_tokens,
    kv_heads, n)` as from `select_pages`: row t's heads of a key head see the keys at or before its position on these pages of its request
    alone (places in its row of `block_table`; others, and -1, stand for nothing; one named twice counts twice); not with `window_size`.
    """
    _check_cache(key_cache, value_cache)
    _check_scales(key_scales, "key_scales", key_cache)
    _check_scales(value_scales, "value_scales", value_cache)
    device, listed = key_cache.device, pages
    pages, page_size, kv_heads, dim = key_cache.shape
    narrow = key_cache.dtype == _E4M3
    if queries.device != device or queries.dtype != key_cache.dtype and not narrow:
        raise ValueError(f"queries must be {key_cache.dtype} on {device}, got {queries.dtype} on {queries.device}")
    if queries.dim() != 3 or queries.shape[2] != dim or queries.stride(2) != 1:
        raise ValueError(f"queries must be (n_tokens, heads, {dim}) with innermost stride 1, got {tuple(queries.shape)}")
    tokens, heads = queries.shape[0], queries.shape[1]
    _check(kv_lens, "kv_lens", torch.int32, None, device)
    n = kv_lens.shape[0]
    _check(cu_new, "cu_new", torch.int32, n + 1, device)
    _check_table(block_table, n, device)
    if sinks is not None:
        _check(sinks, "sinks", torch.float32, heads, device)
    if sink_size < 0 or window_size < 0:
        raise ValueError(f"sink_size and window_size must not be negative, got {sink_size} and {window_size}")
    if sink_size and not window_size:
        raise ValueError("sink_size without window_size: all keys are visible; give both or neither")
    if max_context is not None and max_context < 0:
        raise ValueError(f"max_context must not be negative, got {max_context}")
    if listed is not None:
        if window_size:
            raise ValueError("pages and window_size do not go together")
        if listed.device != device or listed.dtype != torch.int32 or listed.dim() != 3 or listed.shape[:2] != (tokens, kv_heads) \
                or listed.shape[2] == 0 or not listed.is_contiguous():
            raise ValueError(f"pages must be contiguous int32 ({tokens}, {kv_heads}, n) on {device}, got {listed.dtype} {tuple(listed.shape)} on "
                             f"{listed.device}")
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=queries.dtype, device=device)
    elif out.device != device or out.dtype != queries.dtype or out.shape != queries.shape or out.stride(2) != 1:
        raise ValueError(f"out must be {queries.dtype} of shape {tuple(queries.shape)} on {device} with innermost stride 1")
    if narrow or listed is not None:
        args = N.PageAttentionArgs(
            queries.data_ptr(), queries.stride(0), queries.stride(1), _cache_block(key_cache, value_cache, key_scales, value_scales),
            N.PageRequests(block_table.data_ptr(), _pitch(block_table), block_table.shape[1], kv_lens.data_ptr(), cu_new.data_ptr(), n, tokens),
            N.ptr(listed), 0 if listed is None else listed.shape[2], N.ptr(sinks), N.dtype_code(queries.dtype), heads,
            min(max_context or 0, 2 ** 31 - 1), min(sink_size, 2 ** 31 - 1), min(window_size, 2 ** 31 - 1), float(scaling),
            out.data_ptr(), out.stride(0), out.stride(1), None, 0, N.stream_ptr(device))
        size = N.page_work_bytes("attention", args)
        work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        args.work, args.work_bytes = N.ptr(work), size
        N.call_on(device, "sah_page_attention", args)
        return out
    args = N.PagedAttentionArgs(
        queries.data_ptr(), queries.stride(0), queries.stride(1), key_cache.data_ptr(), *key_cache.stride()[:3],
        value_cache.data_ptr(), *value_cache.stride()[:3], block_table.data_ptr(), _pitch(block_table), block_table.shape[1],
        kv_lens.data_ptr(), cu_new.data_ptr(), N.ptr(sinks), N.dtype_code(queries.dtype), n, tokens, heads, kv_heads, dim,
        pages, page_size, min(max_context or 0, 2 ** 31 - 1), min(sink_size, 2 ** 31 - 1), min(window_size, 2 ** 31 - 1), float(scaling),
        out.data_ptr(), out.stride(0), out.stride(1), None, 0, N.stream_ptr(device))
    floats = N.paged_work_floats(args)
    work = torch.empty(floats, dtype=torch.float32, device=device) if floats else None
    args.work, args.work_floats = N.ptr(work), floats
    N.call_on(device, "sah_paged_attention", args)
    return out


def load_paged(key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, length: int, *,
               dtype: Optional[torch.dtype] = None, key_scales: Optional[torch.Tensor] = None,
               value_scales: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The requests' contexts as two contiguous tensors `(n_requests, kv_heads, length, head_dim)`: keys and values at positions below
    `kv_lens[b]`, 0 behind them and on pages that are not there. `dtype`: of an 8-bit cache float32, bfloat16 (default; exact, as float32) or
    float16 (which ends at its largest number, +-65504); of others their own. Addresses and strides multiples of 16 bytes, page_size a power of two."""
    _check_cache(key_cache, value_cache)
    _check_scales(key_scales, "key_scales", key_cache)
    _check_scales(value_scales, "value_scales", value_cache)
    device = key_cache.device
    _check(kv_lens, "kv_lens", torch.int32, None, device)
    n = kv_lens.shape[0]
    _check_table(block_table, n, device)
    narrow = key_cache.dtype == _E4M3
    dtype = (torch.bfloat16 if narrow else key_cache.dtype) if dtype is None else dtype
    if not narrow and dtype != key_cache.dtype:
        raise ValueError(f"dtype of a {key_cache.dtype} cache must be that, got {dtype}")
    if not 0 <= length < 2 ** 31:
        raise ValueError(f"length must be in [0, 2^31), got {length}")
    code, shape = N.dtype_code(dtype), (n, key_cache.shape[2], length, key_cache.shape[3])
    keys, values = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
    if n:
        N.call_on(device, "sah_page_load", N.PageLoadArgs(
            _cache_block(key_cache, value_cache, key_scales, value_scales),
            N.PageRequests(block_table.data_ptr(), _pitch(block_table), block_table.shape[1], kv_lens.data_ptr(), None, n, 0),
            keys.data_ptr(), values.data_ptr(), code, length, N.stream_ptr(device)))
    return keys, values


def _check_bounds(bounds: torch.Tensor, pages: int, kv_heads: int, dim: int, dtype: torch.dtype, device: torch.device) -> None:
    if bounds.device != device or bounds.dtype != dtype or bounds.shape != (pages, kv_heads, 2, dim) or not bounds.is_contiguous():
        raise ValueError(f"bounds must be contiguous {dtype} ({pages}, {kv_heads}, 2, {dim}) on {device}, got {bounds.dtype} {tuple(bounds.shape)} "
                         f"on {bounds.device}")


def update_page_bounds(bounds: torch.Tensor, key_cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, cu_new: torch.Tensor, *,
                       key_scales: Optional[torch.Tensor] = None) -> None:
    """Brings `bounds` `(n_pages, kv_heads, 2, head_dim)`, the smallest and the largest element of each channel of a page's keys, up to date after
    a step's keys have been stored: for the pages whose last token is one of the step's. The others' stay as they were (a page that is not
    full is its tokens' own, which every selection takes). The cache's type; bfloat16 for an 8-bit one, which is exact. A channel with a NaN has
    NaN."""
    _check_cache(key_cache, key_cache)
    _check_scales(key_scales, "key_scales", key_cache)
    device = key_cache.device
    pages, page_size, heads, dim = key_cache.shape
    _check_bounds(bounds, pages, heads, dim, torch.bfloat16 if key_cache.dtype == _E4M3 else key_cache.dtype, device)
    _check(kv_lens, "kv_lens", torch.int32, None, device)
    n = kv_lens.shape[0]
    _check(cu_new, "cu_new", torch.int32, n + 1, device)
    _check_table(block_table, n, device)
    N.call_on(device, "sah_page_bounds", N.PageBoundsArgs(
        _cache_block(key_cache, None, key_scales, None),
        N.PageRequests(block_table.data_ptr(), _pitch(block_table), block_table.shape[1], kv_lens.data_ptr(), cu_new.data_ptr(), n, 0),
        bounds.data_ptr(), N.stream_ptr(device)))


def select_pages(queries: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, cu_new: torch.Tensor,
                 page_size: int, n_select: int, *, sink_pages: int = 1, window_pages: int = 1, max_context: Optional[int] = None) -> torch.Tensor:
    """The pages that each new token attends to, one list for each key head: int32 `(n_tokens, kv_heads, n_select)`, places in the
    request's row of `block_table`, rising, -1 behind the last.

    Of the pages at or before the token's own: the first `sink_pages`, the last `window_pages` (at least 1, its own), and of the others as many as
    make `n_select` with the largest `sum over the key head's query heads and over channels of max(q * smallest, q * largest)`, the most
    that the heads' products with a key of the page can come to together; ties to the lower page, scores that are not finite first. Scores are
    held in 64 bits and summed in one order: results repeat, and only scores within 4 head_dim * 2^-53 of the sum of their terms' sizes may rank either way. Pages that are not there are no candidates. `bounds` as
    `update_page_bounds` keeps them. `max_context` as for `paged_attention`.
    """
    N.require_device(queries, "queries")
    device = queries.device
    if queries.dim() != 3 or queries.stride(2) != 1 and queries.shape[2] > 1:
        raise ValueError(f"queries must be (n_tokens, heads, head_dim) with innermost stride 1, got {tuple(queries.shape)}")
    tokens, heads, dim = queries.shape
    pages, kv_heads = (bounds.shape[0], bounds.shape[1]) if bounds.dim() == 4 else (-1, -1)
    _check_bounds(bounds, pages, kv_heads, dim, bounds.dtype, device)
    _check(kv_lens, "kv_lens", torch.int32, None, device)
    n = kv_lens.shape[0]
    _check(cu_new, "cu_new", torch.int32, n + 1, device)
    _check_table(block_table, n, device)
    _check_page_size(page_size)
    if max_context is not None and max_context < 0:
        raise ValueError(f"max_context must not be negative, got {max_context}")
    if sink_pages < 0 or window_pages < 1 or not sink_pages + window_pages <= n_select < 2 ** 31:
        raise ValueError(f"select_pages needs sink_pages >= 0, window_pages >= 1 and n_select of at least their sum, got {sink_pages}, {window_pages}, {n_select}")
    chosen = torch.empty((tokens, kv_heads, n_select), dtype=torch.int32, device=device)
    args = N.PageSelectArgs(
        queries.data_ptr(), queries.stride(0), queries.stride(1), bounds.data_ptr(), N.dtype_code(queries.dtype), N.dtype_code(bounds.dtype),
        heads, kv_heads, dim, pages, page_size,
        N.PageRequests(block_table.data_ptr(), _pitch(block_table), block_table.shape[1], kv_lens.data_ptr(), cu_new.data_ptr(), n, tokens),
        n_select, sink_pages, window_pages, min(max_context or 0, 2 ** 31 - 1), chosen.data_ptr(), None, 0, N.stream_ptr(device))
    size = N.page_work_bytes("select", args)
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    args.work, args.work_bytes = N.ptr(work), size
    N.call_on(device, "sah_page_select", args)
    return chosen


class PagedKVCache:
    """The caches of `n_layers` layers and the state of up to `n_requests` requests of up to `max_context` tokens each.

        cache = PagedKVCache(n_layers, n_pages, page_size, kv_heads, head_dim, n_requests, max_context, dtype, device)
        step = cache.assign(new_lens, n_tokens)
        for layer ...: out = cache.attend(layer, queries, keys, values, step, scaling)
        cache.release(finished)

    `dtype=torch.float8_e4m3fn` holds keys and values in 8 bits, with scales. `page_bounds=True` keeps the bounds of pages, by which `attend(...,
    n_select=)` lets every token read that many pages only.
    """

    def __init__(self, n_layers: int, n_pages: int, page_size: int, kv_heads: int, head_dim: int, n_requests: int, max_context: int,
                 dtype: torch.dtype, device: torch.device, page_bounds: bool = False) -> None:
        if min(n_layers, n_pages, page_size, kv_heads, head_dim, n_requests, max_context) <= 0:
            raise ValueError("PagedKVCache needs positive sizes")
        if page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two, got {page_size}")
        narrow = dtype == _E4M3
        if not narrow:
            N.dtype_code(dtype)
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.page_size, self.n_pages, self.max_context = page_size, n_pages, max_context
        shape = (n_layers, n_pages, page_size, kv_heads, head_dim)
        self.key_cache = torch.empty(shape, dtype=dtype, device=device)
        self.value_cache = torch.empty(shape, dtype=dtype, device=device)
        scales = (n_layers, n_pages, kv_heads, page_size)
        self.key_scales = torch.empty(scales, dtype=_E8M0, device=device) if narrow else None
        self.value_scales = torch.empty(scales, dtype=_E8M0, device=device) if narrow else None
        self.bounds = torch.empty((n_layers, n_pages, kv_heads, 2, head_dim), dtype=torch.bfloat16 if narrow else dtype,
                                  device=device) if page_bounds else None
        self.block_table = torch.full((n_requests, -(-max_context // page_size)), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(n_requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device)  # page 0 is taken first
        self.free_count = torch.full((1,), n_pages, dtype=torch.int32, device=device)

    def _layer(self, layer: int) -> dict:
        if self.key_scales is None:
            return {}
        return dict(key_scales=self.key_scales[layer], value_scales=self.value_scales[layer])

    def assign(self, new_lens: torch.Tensor, n_tokens: int) -> PageAssignment:
        """`assign_pages` on this cache's state."""
        return assign_pages(new_lens, self.lens, self.block_table, self.free_pages, self.free_count, self.page_size, n_tokens)

    def attend(self, layer: int, queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, step: PageAssignment, scaling: float, *,
               n_select: Optional[int] = None, sink_pages: int = 1, window_pages: int = 1, **options) -> torch.Tensor:
        """`store_paged`, then `paged_attention` (whose keyword arguments `options` are), for one layer. With `page_bounds` the pages' bounds are
        kept, and `n_select` attends to the pages of `select_pages`."""
        if n_select is not None and self.bounds is None:
            raise ValueError("n_select needs a PagedKVCache with page_bounds=True")
        held = self._layer(layer)
        store_paged(keys, values, self.key_cache[layer], self.value_cache[layer], step.slot_map, **held)
        options.setdefault("max_context", self.max_context)
        if self.bounds is not None:
            update_page_bounds(self.bounds[layer], self.key_cache[layer], self.block_table, step.kv_lens, step.cu_new,
                               key_scales=held.get("key_scales"))
            if n_select is not None:
                options["pages"] = select_pages(queries, self.bounds[layer], self.block_table, step.kv_lens, step.cu_new, self.page_size, n_select,
                                                sink_pages=sink_pages, window_pages=window_pages, max_context=options["max_context"])
        return paged_attention(queries, self.key_cache[layer], self.value_cache[layer], self.block_table, step.kv_lens, step.cu_new,
                               scaling, **held, **options)

    def load(self, layer: int, length: int, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """`load_paged` of one layer: all requests' contexts, `(n_requests, kv_heads, length, head_dim)`."""
        return load_paged(self.key_cache[layer], self.value_cache[layer], self.block_table, self.lens, length, dtype=dtype, **self._layer(layer))

    def release(self, finished: torch.Tensor) -> None:
        """`release_pages` on this cache's state."""
        release_pages(finished, self.lens, self.block_table, self.free_pages, self.free_count, self.page_size)
