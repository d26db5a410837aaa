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
"""
from __future__ import annotations

from typing import NamedTuple, Optional

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
                slot_map: torch.Tensor) -> None:
    """Writes `keys[t]` and `values[t]`, `(n_tokens, kv_heads, head_dim)`, to slot `slot_map[t]` of the caches; rows with a slot of -1
    (or any other outside the cache) are passed over. No two rows may name the same slot: which of them it would hold is
    not defined."""
    _check_cache(key_cache, value_cache)
    device = key_cache.device
    pages, page_size, heads, dim = key_cache.shape
    rows, dtype = (keys.shape[0] if keys.dim() else 0, heads, dim), key_cache.dtype
    for t, what in ((keys, "keys"), (values, "values")):
        if t.device != device or t.dtype != dtype:
            raise ValueError(f"{what} must be {dtype} on {device}, got {t.dtype} on {t.device}")
        if t.shape != rows:
            raise ValueError(f"{what} must have shape (n_tokens, {heads}, {dim}), got {tuple(t.shape)}")
        if t.stride(2) != 1 and dim > 1:
            raise ValueError(f"{what}: the innermost stride must be 1")
    _check(slot_map, "slot_map", torch.int64, rows[0], device)
    N.call_on(device, "sah_paged_store", N.PagedStoreArgs(
        keys.data_ptr(), keys.stride(0), keys.stride(1), values.data_ptr(), values.stride(0), values.stride(1),
        key_cache.data_ptr(), *key_cache.stride()[:3], value_cache.data_ptr(), *value_cache.stride()[:3],
        slot_map.data_ptr(), N.dtype_code(dtype), rows[0], heads, dim, pages, page_size, N.stream_ptr(device)))


def paged_attention(queries: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, cu_new: torch.Tensor, scaling: float, *, max_context: Optional[int] = None,
                    sink_size: int = 0, window_size: int = 0, sinks: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of packed new tokens `(n_tokens, heads, head_dim)` over the cache, which holds their keys already.

    Row `cu_new[b] + i` stands at position `kv_lens[b] - new_b + i` of request b, `new_b = cu_new[b + 1] - cu_new[b]`, and sees the request's
    keys up to its own; with `window_size > 0` of those only the first `sink_size` and the last `window_size`, the columns of
    `SinkMasker` and `LocalMasker`. `sinks` (float32 `(heads,)`): a logit per head in the denominator. Query heads share key heads in
    groups, as `repeat_kv` would have it. A row that sees nothing is 0; rows behind the last request's keep what `out` held (without
    `out`: unspecified). `max_context`, about the longest request's length, decides how work is split (default: the
    table's width); results do not depend on it beyond the order of sums. head_dim a multiple of 8 up to 256, page_size a power of two,
    addresses and strides multiples of 16 bytes; `out` shares no memory with the other tensors (refused; it and
    the queries may be slices of one buffer, their tokens equally far apart). Returns `(n_tokens, heads, head_dim)`.
    """
    _check_cache(key_cache, value_cache)
    device = key_cache.device
    pages, page_size, kv_heads, dim = key_cache.shape
    if queries.device != device or queries.dtype != key_cache.dtype:
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
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=queries.dtype, device=device)
    elif out.device != device or out.dtype != queries.dtype or out.shape != queries.shape or out.stride(2) != 1:
        raise ValueError(f"out must be {queries.dtype} of shape {tuple(queries.shape)} on {device} with innermost stride 1")
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


class PagedKVCache:
    """The caches of `n_layers` layers and the state of up to `n_requests` requests of up to `max_context` tokens each.

        cache = PagedKVCache(n_layers, n_pages, page_size, kv_heads, head_dim, n_requests, max_context, dtype, device)
        step = cache.assign(new_lens, n_tokens)
        for layer ...: out = cache.attend(layer, queries, keys, values, step, scaling)
        cache.release(finished)
    """

    def __init__(self, n_layers: int, n_pages: int, page_size: int, kv_heads: int, head_dim: int, n_requests: int, max_context: int,
                 dtype: torch.dtype, device: torch.device) -> None:
        if min(n_layers, n_pages, page_size, kv_heads, head_dim, n_requests, max_context) <= 0:
            raise ValueError("PagedKVCache needs positive sizes")
        if page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two, got {page_size}")
        N.dtype_code(dtype)
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.page_size, self.n_pages, self.max_context = page_size, n_pages, max_context
        shape = (n_layers, n_pages, page_size, kv_heads, head_dim)
        self.key_cache = torch.empty(shape, dtype=dtype, device=device)
        self.value_cache = torch.empty(shape, dtype=dtype, device=device)
        self.block_table = torch.full((n_requests, -(-max_context // page_size)), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(n_requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device)  # page 0 is taken first
        self.free_count = torch.full((1,), n_pages, dtype=torch.int32, device=device)

    def assign(self, new_lens: torch.Tensor, n_tokens: int) -> PageAssignment:
        """`assign_pages` on this cache's state."""
        return assign_pages(new_lens, self.lens, self.block_table, self.free_pages, self.free_count, self.page_size, n_tokens)

    def attend(self, layer: int, queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, step: PageAssignment, scaling: float,
               **options) -> torch.Tensor:
        """`store_paged`, then `paged_attention` (whose keyword arguments `options` are), for one layer."""
        store_paged(keys, values, self.key_cache[layer], self.value_cache[layer], step.slot_map)
        options.setdefault("max_context", self.max_context)
        return paged_attention(queries, self.key_cache[layer], self.value_cache[layer], self.block_table, step.kv_lens, step.cu_new,
                               scaling, **options)

    def release(self, finished: torch.Tensor) -> None:
        """`release_pages` on this cache's state."""
        release_pages(finished, self.lens, self.block_table, self.free_pages, self.free_count, self.page_size)
