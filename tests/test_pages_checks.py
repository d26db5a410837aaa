"""include/sah_pages.h on the host: exports, layouts, argument checks of the C entry points and of the Python functions (no GPU)."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

from sparse_attention_hub_amd import _native as N
from sparse_attention_hub_amd.sparse_attention.utils import paged_cache as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_BUF = ctypes.create_string_buffer(4096)  # stands for device memory: never dereferenced by the checks
_PTR = (ctypes.addressof(_BUF) + 63) // 64 * 64
_FAR = 2 ** 40  # no two multiples of it are near each other, and none is dereferenced
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _call(name, args, **changes):
    for path, value in changes.items():
        at = args
        *outer, field = path.split("__")
        for name_ in outer:
            at = getattr(at, name_)
        assert hasattr(at, field), path
        setattr(at, field, value)
    lib = N.lib()
    rc = getattr(lib, name)(ctypes.byref(args))
    assert rc == 0 or name.encode() in lib.sah_last_error()
    return rc


def _cache(dtype=N.SAH_E4M3, k=_FAR, v=2 * _FAR):
    # 8 pages of 16 tokens, 2 heads of 64
    return N.PageCache(k, 2048, 128, 64, v, 2048, 128, 64, 3 * _FAR, 4 * _FAR, dtype, 8, 16, 2, 64)


def _requests():
    return N.PageRequests(5 * _FAR, 4, 4, 6 * _FAR, 7 * _FAR, 1, 3)


def test_every_declared_symbol_is_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "sah_pages.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(?:int|int64_t)\s+(sah_\w+)\s*\(", text))
    assert declared == set(N.PAGE_SYMBOLS) | set(N.PAGE_SIZE_SYMBOLS)
    lib = N.lib()
    for fn in N.PAGE_SYMBOLS:
        assert getattr(lib, fn)(None) == -2 and fn.encode() in lib.sah_last_error(), fn
    for fn in N.PAGE_SIZE_SYMBOLS:
        assert getattr(lib, fn)(None) == 0
    assert int(re.search(r"#define SAH_E4M3 (\d+)", text).group(1)) == N.SAH_E4M3


def test_argument_blocks_are_laid_out_as_in_the_header(tmp_path):
    """Field offsets of the ctypes structures against the C compiler's."""
    structs = {"sah_page_cache": N.PageCache, "sah_page_requests": N.PageRequests, "sah_page_store_args": N.PageStoreArgs,
               "sah_page_load_args": N.PageLoadArgs, "sah_page_bounds_args": N.PageBoundsArgs, "sah_page_select_args": N.PageSelectArgs,
               "sah_page_attention_args": N.PageAttentionArgs}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "sah_pages.h"', "int main(void) {"]
    want = []
    for name, cls in structs.items():
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in got] == want


_CACHE_REFUSALS = [
    (dict(cache__dtype=4), -5), (dict(cache__dtype=-1), -5), (dict(cache__n_pages=0), -1), (dict(cache__Hkv=0), -1), (dict(cache__D=72), -3),
    (dict(cache__D=0), -3), (dict(cache__D=272), -3), (dict(cache__page_size=24), -3), (dict(cache__page_size=0), -3), (dict(cache__k=None), -2),
    (dict(cache__k_scales=None), -2), (dict(cache__k=_FAR + 8), -1), (dict(cache__ks_t=129), -1), (dict(cache__ks_h=72), -1),
    (dict(cache__k_scales=_FAR + 2), -1), (dict(cache__ks_t=2 ** 26), -3), (dict(cache__ks_t=-64), -3),
]
_VALUE_REFUSALS = [(dict(cache__v=None), -2), (dict(cache__v_scales=None), -2), (dict(cache__vs_p=2049), -1), (dict(cache__vs_t=2 ** 27), -3)]
_REQUEST_REFUSALS = [
    (dict(requests__n_requests=0), -1), (dict(requests__table_width=0), -1), (dict(requests__table_pitch=3), -1), (dict(requests__block_table=None), -2),
    (dict(requests__kv_lens=None), -2), (dict(requests__table_width=2 ** 27, requests__table_pitch=2 ** 27), -3),
]
_ROW_REFUSALS = [(dict(requests__cu_new=None), -2)]


@pytest.mark.parametrize("changes, code", _CACHE_REFUSALS + _VALUE_REFUSALS + [
    (dict(cache__dtype=1), -5), (dict(dtype=3), -5), (dict(n_tokens=-1), -1), (dict(k=None), -2), (dict(v=None), -2), (dict(slot_map=None), -2), (dict(k=8 * _FAR + 8), -1),
    (dict(ks_t=129), -1), (dict(vs_h=60), -1), (dict(cache__ks_p=0), -1), (dict(cache__vs_t=48), -1), (dict(cache__ks_h=32), -1),
    (dict(n_tokens=2 ** 31 - 1, cache__Hkv=2 ** 10, cache__ks_t=2 ** 17, cache__ks_p=2 ** 21, cache__vs_t=2 ** 17, cache__vs_p=2 ** 21), -3),
])
def test_store_refuses(changes, code):
    args = N.PageStoreArgs(_cache(), 8 * _FAR, 128, 64, 9 * _FAR, 128, 64, 10 * _FAR, 1, 3, None)
    assert _call("sah_page_store", args, **changes) == code


@pytest.mark.parametrize("changes, code", _CACHE_REFUSALS + _VALUE_REFUSALS + _REQUEST_REFUSALS + [
    (dict(dtype=3), -5), (dict(cache__dtype=1, dtype=2), -5), (dict(length=-1), -1), (dict(k_out=None), -2), (dict(v_out=None), -2), (dict(v_out=_FAR + 8), -1),
    (dict(length=2 ** 31 - 1, requests__n_requests=2 ** 20), -3),
])
def test_load_refuses(changes, code):
    args = N.PageLoadArgs(_cache(), _requests(), 8 * _FAR, 9 * _FAR, 1, 40, None)
    assert _call("sah_page_load", args, **changes) == code


@pytest.mark.parametrize("changes, code", _CACHE_REFUSALS + _REQUEST_REFUSALS + _ROW_REFUSALS + [(dict(bounds=None), -2), (dict(bounds=_FAR + 8), -1)])
def test_bounds_refuse(changes, code):
    args = N.PageBoundsArgs(_cache(v=None), _requests(), 8 * _FAR, None)
    assert _call("sah_page_bounds", args, **changes) == code


@pytest.mark.parametrize("changes, code", _REQUEST_REFUSALS + _ROW_REFUSALS + [
    (dict(dtype=3), -5), (dict(bounds_dtype=3), -5), (dict(Hq=3), -1), (dict(Hkv=0), -1), (dict(n_pages=0), -1), (dict(max_context=-1), -1), (dict(D=60), -3),
    (dict(D=264), -3), (dict(page_size=3), -3), (dict(n_select=2), -1), (dict(sink_pages=-1), -1), (dict(window_pages=0), -1),
    (dict(sink_pages=2 ** 31 - 1, window_pages=2 ** 31 - 1), -1), (dict(q=None), -2), (dict(bounds=None), -2), (dict(pages=None), -2), (dict(bounds=_FAR + 4), -1), (dict(q=_FAR + 8), -1), (dict(qs_t=260), -1), (dict(qs_h=68), -1),
    (dict(work=None), -4), (dict(work_bytes=100), -4), (dict(work=_FAR + 8), -4), (dict(requests__n_tokens=-1), -1),
    (dict(requests__n_tokens=2 ** 30, work_bytes=2 ** 60), -3),
])
def test_select_refuses(changes, code):
    args = N.PageSelectArgs(8 * _FAR, 256, 64, 9 * _FAR, 1, 1, 4, 2, 64, 8, 16, _requests(), 3, 1, 2, 0, 10 * _FAR, 11 * _FAR, 2 ** 20, None)
    assert _call("sah_page_select", args, **changes) == code


def _attention(**changes):
    args = N.PageAttentionArgs(8 * _FAR, 256, 64, _cache(), _requests(), None, 0, None, 1, 4, 0, 0, 0, 0.125, 9 * _FAR, 256, 64, 10 * _FAR, 2 ** 40, None)
    return _call("sah_page_attention", args, **changes)


@pytest.mark.parametrize("changes, code", _CACHE_REFUSALS + _VALUE_REFUSALS + _REQUEST_REFUSALS + _ROW_REFUSALS + [
    (dict(dtype=3), -5), (dict(cache__dtype=2), -5), (dict(cache__dtype=1), -5), (dict(Hq=3), -1), (dict(Hq=0), -1), (dict(max_context=-1), -1),
    (dict(sink=-1), -1), (dict(window=-1), -1), (dict(n_select=-1), -1), (dict(n_select=4), -1), (dict(pages=11 * _FAR), -1),
    (dict(pages=11 * _FAR, n_select=3, window=4), -1), (dict(pages=11 * _FAR, n_select=3, sink=4), -1), (dict(pages=11 * _FAR, n_select=2 ** 27), -3),
    (dict(requests__n_tokens=2 ** 29), -3), (dict(requests__n_tokens=-1), -1), (dict(q=None), -2), (dict(out=None), -2), (dict(q=8 * _FAR + 2), -1),
    (dict(qs_h=60), -1), (dict(os_t=257), -1), (dict(work=10 * _FAR + 8), -1), (dict(os_t=0), -1), (dict(os_h=32), -1), (dict(scaling=math.nan), -1),
    (dict(scaling=math.inf), -1), (dict(work=None, requests__n_tokens=60), -4), (dict(work_bytes=64, requests__n_tokens=60), -4),
    (dict(work=None, requests__table_width=1000, requests__table_pitch=1000), -4), (dict(work_bytes=64, requests__table_width=1000, requests__table_pitch=1000), -4),
    (dict(out=8 * _FAR), -1), (dict(out=_FAR + 32), -1), (dict(out=2 * _FAR), -1), (dict(out=3 * _FAR), -1), (dict(out=4 * _FAR + 240), -1), (dict(out=5 * _FAR), -1),
    (dict(out=6 * _FAR), -1), (dict(out=7 * _FAR), -1), (dict(out=11 * _FAR, pages=11 * _FAR, n_select=3), -1), (dict(out=12 * _FAR, sinks=12 * _FAR), -1),
])
def test_attention_refuses(changes, code):
    assert _attention(**changes) == code


@pytest.mark.parametrize("changes", [
    dict(requests__n_tokens=1, qs_t=257, os_t=3), dict(cache__n_pages=1, cache__ks_p=2049, cache__vs_p=-1), dict(cache__page_size=1, cache__ks_t=2 ** 40 + 1, cache__vs_t=-3),
    dict(Hq=1, cache__Hkv=1, qs_h=65, cache__ks_h=3, cache__vs_h=5, os_h=-1),
])
def test_any_stride_of_a_dimension_of_one_entry_is_taken(changes):
    """What is refused is the workspace that is not given."""
    assert _attention(work=None, requests__table_width=4000, requests__table_pitch=4000, **changes) == -4


def test_nothing_to_do_is_no_error():
    assert _call("sah_page_store", N.PageStoreArgs(cache=_cache())) == 0
    assert _call("sah_page_load", N.PageLoadArgs(_cache(), _requests(), None, None, 1, 0, None)) == 0
    assert _attention(requests__n_tokens=0, q=None, out=None, work=None) == 0
    args = N.PageSelectArgs(None, 256, 64, None, 1, 1, 4, 2, 64, 8, 16, _requests(), 3, 1, 2, 0, None, None, 0, None)
    assert _call("sah_page_select", args, requests__n_tokens=0) == 0


@pytest.mark.parametrize("page_size, ok", [(1, True), (2, True), (4, True), (8, True), (16, False), (64, False)])
def test_scales_of_small_pages_may_begin_anywhere(page_size, ok):
    """A layer's scales are a slice of all layers': where its pages hold few tokens, it begins at any byte."""
    for offset in (1, 2, 3):
        changes = dict(cache__page_size=page_size, cache__k_scales=3 * _FAR + offset, cache__v_scales=4 * _FAR + offset)
        # nothing to do, or a refusal that comes behind those of the cache
        store = N.PageStoreArgs(_cache(), 8 * _FAR, 128, 64, 9 * _FAR, 128, 64, 10 * _FAR, 1, 0, None)
        assert _call("sah_page_store", store, **changes) == (0 if ok else -1)
        load = N.PageLoadArgs(_cache(), _requests(), 8 * _FAR, 9 * _FAR, 1, 0, None)
        assert _call("sah_page_load", load, **changes) == (0 if ok else -1)
        assert _call("sah_page_bounds", N.PageBoundsArgs(_cache(v=None), _requests(), None, None), **changes) == (-2 if ok else -1)
        assert _attention(requests__n_tokens=0, **changes) == (0 if ok else -1)


@pytest.mark.parametrize("dtype", [N.SAH_E4M3, 1])
def test_lists_of_no_tokens_are_no_error(dtype):
    """An empty tensor has no address."""
    nothing = dict(requests__n_tokens=0, q=None, out=None, work=None, cache__dtype=dtype)
    assert _attention(n_select=4, pages=None, **nothing) == 0 and _attention(n_select=4, pages=11 * _FAR, **nothing) == 0
    assert _attention(n_select=4, pages=None, window=4, **nothing) == -1 and _attention(n_select=0, pages=11 * _FAR, **nothing) == -1


def test_workspaces_follow_the_work():
    def attention(tokens, width, requests=1, n_select=0, Hq=8):
        args = N.PageAttentionArgs(dtype=1, Hq=Hq, n_select=n_select, pages=_PTR if n_select else None, cache=N.PageCache(dtype=3, n_pages=9, page_size=16, Hkv=2, D=128),
                                   requests=N.PageRequests(table_width=width, n_requests=requests, n_tokens=tokens))
        return N.page_work_bytes("attention", args)

    # two parts of 16 rows for each key head of a workgroup, of which there are as many as there is work for, 4 a CU at most
    assert 0 < attention(1, 8) <= attention(1, 64) <= attention(1, 2048) <= attention(1, 2 ** 20) <= 1024 * 2 * 2 * 16 * 132 * 4
    assert attention(1, 1000, n_select=8) <= attention(1, 8) < 2 ** 20
    # a chunk: the contexts in 16 bits, their table, and what the attention over them needs
    copy = 2 * 2 * 2048 * 16 * 2 * 128 + 4 * 2048
    assert copy < attention(2048, 2048) < copy + 2 ** 28
    # no copy of more than 2^33 bytes
    assert attention(2048, 2 ** 20) < 2 ** 33
    select = N.PageSelectArgs(Hkv=2, requests=N.PageRequests(table_width=1000, n_tokens=7))
    assert N.page_work_bytes("select", select) == 7 * 2 * 1000 * 8


@pytest.mark.parametrize("dtype", [1, 2])
def test_the_copy_of_a_chunk_has_room_for_what_the_caller_says(dtype):
    def attention(slots, tokens, max_context, width=8192, page_size=16, n_pages=9):
        args = N.PageAttentionArgs(dtype=dtype, Hq=32, max_context=max_context, cache=N.PageCache(dtype=3, n_pages=n_pages, page_size=page_size, Hkv=8, D=128),
                                   requests=N.PageRequests(table_width=width, n_requests=slots, n_tokens=tokens))
        return N.page_work_bytes("attention", args)

    def copy(slots, pages, page_size=16):
        return slots * (4 * pages * page_size * 8 * 128 + 4 * pages)

    rest = 2 ** 27  # what the kernels need beside it, and what was lost
    for slots, hint in ((1, 4096), (16, 4096), (16, 4081), (16, 5000), (64, 8192)):
        assert copy(slots, -(-hint // 16)) <= attention(slots, 4096, hint) <= copy(slots, -(-hint // 16)) + rest
    assert copy(1, 8192) <= attention(1, 4096, 0) <= copy(1, 8192) + rest        # not said: the table's
    assert copy(1, 8192) <= attention(1, 4096, 2 ** 31 - 1) <= copy(1, 8192) + rest
    assert copy(4, 1, 4096) <= attention(4, 4096, 7, 32, 4096) <= copy(4, 1, 4096) + rest
    # rooms of more than 2 GiB: as many pages as the cache has, 2 GiB at most, and a table
    for slots, hint, width in ((16, 0, 8192), (16, 131072, 8192), (64, 16384, 8192), (2, 2 ** 31 - 1, 2 ** 20)):
        for n_pages in (9, 1000, 30000, 2 ** 22):
            least = 4 * min(n_pages, 2 ** 15) * 16 * 8 * 128
            assert least <= attention(slots, 4096, hint, width, n_pages=n_pages) <= least + rest
    # tables whose copy is more than a launch's workgroups, or whose own table is large: the cache as it is
    assert attention(1024, 40000, 0, 2 ** 12, 4096, 9) <= rest and attention(2 ** 14, 2 ** 20, 0, 2 ** 13, 1, 9) <= rest


def test_the_workspace_of_a_selection_is_bounded():
    def select(tokens, width, Hkv=8):
        return N.page_work_bytes("select", N.PageSelectArgs(Hkv=Hkv, requests=N.PageRequests(table_width=width, n_tokens=tokens)))

    assert select(100, 8192) == 100 * 8 * 8192 * 8
    assert select(512, 8192) == 2 ** 28 == select(513, 8192) == select(2 ** 20, 8192)
    assert 2 ** 28 - 3000 * 8 < select(2 ** 20, 3000) <= 2 ** 28
    assert select(9, 2 ** 26) == 2 ** 29  # a row's keys are a row's


# _cache(): 8 pages of 16 tokens and 2 heads of 64, its scales 256 bytes; _requests(): a table of 4 entries, one length, two sums
@pytest.mark.parametrize("dtype, size", [(0, 4), (1, 2)])
def test_outputs_on_what_a_call_reads_are_refused(dtype, size):
    out = 2 * 40 * 64 * size  # bytes of a context read back
    held = N.PageLoadArgs(_cache(), _requests(), 8 * _FAR, 9 * _FAR, dtype, 40, None)
    ends = [_FAR + 8 * 2048 - 16, 2 * _FAR + 8 * 2048 - 16, 3 * _FAR + 240, 4 * _FAR + 240, 5 * _FAR, 6 * _FAR, _FAR - out + 16]
    for field in ("k_out", "v_out"):
        for at in ends + [8 * _FAR + out - 16 if field == "v_out" else 9 * _FAR - out + 16]:
            assert _call("sah_page_load", N.PageLoadArgs.from_buffer_copy(held), **{field: at}) == -1, at
    for cache_dtype, unit in ((N.SAH_E4M3, 1), (1, 2), (0, 4)):
        whole = 8 * 2 * 2 * 64 * (2 if cache_dtype == N.SAH_E4M3 else unit)  # bytes of bounds
        for at in [_FAR + 8 * 2048 * unit - 16, 5 * _FAR, 6 * _FAR, 7 * _FAR, _FAR - whole + 16] + ([3 * _FAR + 240] if unit == 1 else []):
            assert _call("sah_page_bounds", N.PageBoundsArgs(_cache(v=None, dtype=cache_dtype), _requests(), at, None)) == -1, at

    def select(**changes):  # 3 tokens of 4 heads of 64 in 16 bits, bounds 8 * 2 * 2 * 64
        args = N.PageSelectArgs(8 * _FAR, 256, 64, 9 * _FAR, 1, 1, 4, 2, 64, 8, 16, _requests(), 3, 1, 2, 0, 10 * _FAR, 11 * _FAR, 2 ** 20, None)
        return _call("sah_page_select", args, **changes)

    for at in (8 * _FAR + 3 * 512 - 4, 9 * _FAR + 8 * 2 * 2 * 64 * 2 - 4, 8 * _FAR - 3 * 2 * 3 * 4 + 4, 5 * _FAR + 12, 6 * _FAR, 7 * _FAR + 4):
        assert select(pages=at) == -1, at


def test_tensors_on_the_host_are_refused():
    i32, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    cache = torch.zeros(8, 16, 2, 64).to(_E4M3)
    scales = torch.zeros(8, 2, 16, dtype=torch.uint8).view(_E8M0)
    rows, bounds, cu = torch.zeros(3, 2, 64), torch.zeros(8, 2, 2, 64), torch.zeros(3, dtype=torch.int32)
    held = dict(key_scales=scales, value_scales=scales)
    for call in (lambda: P.store_paged(rows, rows, cache, cache, torch.zeros(3, dtype=torch.int64), **held),
                 lambda: P.load_paged(cache, cache, table, i32, 10, **held),
                 lambda: P.update_page_bounds(bounds, cache, table, i32, cu, key_scales=scales),
                 lambda: P.select_pages(rows, bounds, table, i32, cu, 16, 3),
                 lambda: P.paged_attention(rows, cache, cache, table, i32, cu, 1.0, **held)):
        with pytest.raises(N.NativeLibraryError, match="no CPU fallback"):
            call()


def test_a_cache_in_8_bits_holds_scales_and_bounds():
    cache = P.PagedKVCache(2, 5, 16, 3, 32, 2, 50, _E4M3, "cpu", page_bounds=True)
    assert cache.key_cache.dtype == _E4M3 and cache.key_scales.dtype == _E8M0 and cache.value_scales.shape == (2, 5, 3, 16)
    assert cache.bounds.shape == (2, 5, 3, 2, 32) and cache.bounds.dtype == torch.bfloat16
    cache = P.PagedKVCache(2, 5, 16, 3, 32, 2, 50, torch.float16, "cpu", page_bounds=True)
    assert cache.key_scales is None and cache.bounds.dtype == torch.float16
    cache = P.PagedKVCache(2, 5, 16, 3, 32, 2, 50, torch.float16, "cpu")
    with pytest.raises(ValueError, match="page_bounds"):
        cache.attend(0, None, None, None, None, 1.0, n_select=4)
