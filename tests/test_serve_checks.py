"""include/sah_serve.h on the host: exports, argument checks of the C entry points and of the Python functions (no GPU)."""
import ctypes
import os
import re

import pytest
import torch

from sparse_attention_hub_amd import _native as N
from sparse_attention_hub_amd.sparse_attention.utils import paged_cache as P
from sparse_attention_hub_amd.sparse_attention.utils import token_sampling as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_BUF = ctypes.create_string_buffer(4096)  # stands for device memory: never dereferenced by the checks
_PTR = (ctypes.addressof(_BUF) + 63) // 64 * 64


def _call(name, args):
    lib = N.lib()
    rc = getattr(lib, name)(ctypes.byref(args))
    assert name.encode() in lib.sah_last_error()
    return rc


def _changed(args, changes):
    for name, value in changes.items():
        assert hasattr(args, name)
        setattr(args, name, value)
    return args


def test_every_declared_symbol_is_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "sah_serve.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(?:int|int64_t)\s+(sah_\w+)\s*\(", text))
    assert declared == set(N.SERVE_SYMBOLS) | {"sah_paged_attention_work_floats", "sah_sample_work_bytes"}
    lib = N.lib()
    for fn in N.SERVE_SYMBOLS:
        assert getattr(lib, fn)(None) == -2 and fn.encode() in lib.sah_last_error(), fn
    assert lib.sah_paged_attention_work_floats(None) == 0 and lib.sah_sample_work_bytes(None) == 0


def test_argument_blocks_are_laid_out_as_in_the_header(tmp_path):
    """Field offsets of the ctypes structures against the C compiler's."""
    import subprocess

    structs = {"sah_paged_assign_args": N.PagedAssignArgs, "sah_paged_release_args": N.PagedReleaseArgs,
               "sah_paged_store_args": N.PagedStoreArgs, "sah_paged_attention_args": N.PagedAttentionArgs, "sah_sample_args": N.SampleArgs}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "sah_serve.h"', "int main(void) {"]
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


@pytest.mark.parametrize("changes, code", [
    (dict(n_requests=0), -1), (dict(page_size=0), -1), (dict(table_width=0), -1), (dict(n_pages=0), -1), (dict(n_tokens=-1), -1),
    (dict(n_requests=4097), -3), (dict(table_pitch=3), -1), (dict(new_lens=None), -2), (dict(lens=None), -2), (dict(block_table=None), -2),
    (dict(free_pages=None), -2), (dict(free_count=None), -2), (dict(slot_map=None), -2), (dict(positions=None), -2), (dict(cu_new=None), -2),
    (dict(kv_lens=None), -2), (dict(granted=None), -2), (dict(lens_out=None), -2), (dict(free_count_out=None), -2), (dict(work=None), -2),
    (dict(n_tokens=2 ** 30 + 1), -3),
])
def test_assign_refuses(changes, code):
    args = N.PagedAssignArgs(_PTR, _PTR, _PTR, 4, 4, _PTR, _PTR, 8, 2, 16, 5, _PTR, _PTR, _PTR, _PTR, _PTR, _PTR, _PTR, _PTR, None)
    assert _call("sah_paged_assign", _changed(args, changes)) == code


@pytest.mark.parametrize("changes, code", [
    (dict(n_requests=0), -1), (dict(page_size=0), -1), (dict(table_width=0), -1), (dict(n_pages=0), -1), (dict(n_requests=4097), -3),
    (dict(table_pitch=3), -1), (dict(finished=None), -2), (dict(lens=None), -2), (dict(block_table=None), -2), (dict(free_pages=None), -2),
    (dict(free_count=None), -2), (dict(work=None), -2),
])
def test_release_refuses(changes, code):
    args = N.PagedReleaseArgs(_PTR, _PTR, _PTR, 4, 4, _PTR, _PTR, 8, 2, 16, _PTR, None)
    assert _call("sah_paged_release", _changed(args, changes)) == code


@pytest.mark.parametrize("changes, code", [
    (dict(dtype=3), -5), (dict(n_tokens=-1), -1), (dict(Hkv=0), -1), (dict(D=0), -1), (dict(n_pages=0), -1), (dict(page_size=0), -1),
    (dict(k=None), -2), (dict(v=None), -2), (dict(k_cache=None), -2), (dict(v_cache=None), -2), (dict(slot_map=None), -2),
    (dict(n_tokens=2 ** 31 - 1, Hkv=2 ** 12, kcs_t=2 ** 17, kcs_p=2 ** 21, vcs_t=2 ** 17, vcs_p=2 ** 21), -3),
    (dict(kcs_p=0), -1), (dict(vcs_t=63), -1), (dict(vcs_h=31), -1), (dict(kcs_p=-1024), -1),
])
def test_store_refuses(changes, code):
    args = N.PagedStoreArgs(_PTR, 64, 32, _PTR, 64, 32, _PTR, 1024, 64, 32, _PTR, 1024, 64, 32, _PTR, 1, 3, 2, 32, 4, 16, None)
    assert _call("sah_paged_store", _changed(args, changes)) == code


@pytest.mark.parametrize("changes, code", [
    (dict(dtype=-1), -5), (dict(n_requests=0), -1), (dict(n_tokens=-1), -1), (dict(Hq=3), -1), (dict(Hkv=0), -1), (dict(n_pages=0), -1),
    (dict(table_width=0), -1), (dict(max_context=-1), -1), (dict(sink=-1), -1), (dict(window=-1), -1), (dict(D=60), -3), (dict(D=264), -3),
    (dict(D=0), -3), (dict(page_size=24), -3), (dict(page_size=0), -3), (dict(table_width=2 ** 28, table_pitch=2 ** 28), -3),
    (dict(table_pitch=3), -1), (dict(q=None), -2), (dict(k=None), -2), (dict(v=None), -2), (dict(block_table=None), -2),
    (dict(kv_lens=None), -2), (dict(cu_new=None), -2), (dict(out=None), -2), (dict(q=_PTR + 2), -1), (dict(k=_PTR + 8), -1), (dict(ks_t=129), -1),
    (dict(qs_h=65), -1), (dict(ks_t=2 ** 26), -3), (dict(vs_t=-64), -3), (dict(os_t=257), -1), (dict(scaling=float("nan")), -1),
    (dict(os_t=0), -1), (dict(os_h=0), -1), (dict(os_h=-64), -1), (dict(table_width=2 ** 27 - 255, table_pitch=2 ** 27), -3),
])
def test_attention_refuses(changes, code):
    args = N.PagedAttentionArgs(_PTR, 256, 64, _PTR, 2048, 128, 64, _PTR, 2048, 128, 64, _PTR, 4, 4, _PTR, _PTR, None, 1, 2, 3, 4, 2, 64, 8, 16,
                                0, 0, 0, 0.125, _PTR, 256, 64, _PTR, 0, None)
    assert _call("sah_paged_attention", _changed(args, changes)) == code


@pytest.mark.parametrize("changes", [
    dict(n_tokens=1, qs_t=257, os_t=3), dict(n_pages=1, ks_p=2049, vs_p=-1), dict(page_size=1, ks_t=2 ** 40 + 1, vs_t=-3),
    dict(Hq=1, Hkv=1, qs_h=65, ks_h=3, vs_h=5, os_h=-1),
])
def test_attention_takes_any_stride_of_a_dimension_of_one_entry(changes):
    """Such a dimension's stride is no address: what is refused is the workspace that is not given."""
    args = N.PagedAttentionArgs(_PTR, 256, 64, _PTR, 2048, 128, 64, _PTR, 2048, 128, 64, _PTR, 4, 4, _PTR, _PTR, None, 1, 2, 3, 4, 2, 64, 8, 16,
                                0, 0, 0, 0.125, _PTR, 256, 64, None, 0, None)
    assert _call("sah_paged_attention", _changed(args, changes)) == -4


_FAR = 2 ** 40  # no two of these addresses are near each other, and none is dereferenced


@pytest.mark.parametrize("changes, what", [
    (dict(out=_FAR), b"with q"), (dict(out=_FAR + 2 * 256 * 2), b"with q"), (dict(out=_FAR - 2 * 256 * 2), b"with q"),
    (dict(out=_FAR + 3 * 64 * 2), b"with q"), (dict(out=_FAR + 112), b"with q"), (dict(out=_FAR, os_h=192, os_t=64, qs_h=192, qs_t=64), b"with q"),
    (dict(out=_FAR + 64 * 2, os_t=512), b"with q"), (dict(out=_FAR + 128, n_tokens=1), b"with q"),
    (dict(out=2 * _FAR), b"within"), (dict(out=2 * _FAR + 8 * 2048 * 2 - 16), b"within"), (dict(out=3 * _FAR - 16), b"within"),
    (dict(out=4 * _FAR + 16), b"within"), (dict(out=5 * _FAR), b"within"), (dict(out=6 * _FAR), b"within"), (dict(out=7 * _FAR - 256), b"within"),
])
def test_attention_refuses_an_output_on_what_is_read(changes, what):
    args = N.PagedAttentionArgs(_FAR, 256, 64, 2 * _FAR, 2048, 128, 64, 3 * _FAR, 2048, 128, 64, 4 * _FAR, 4, 4, 5 * _FAR, 6 * _FAR, 7 * _FAR, 1, 2, 3, 4, 2,
                                64, 8, 16, 0, 0, 0, 0.125, 8 * _FAR, 256, 64, 9 * _FAR, 2 ** 40, None)
    assert _call("sah_paged_attention", _changed(args, changes)) == -1
    assert what in N.lib().sah_last_error()


@pytest.mark.parametrize("changes, code", [
    (dict(dtype=7), -5), (dict(n_rows=-1), -1), (dict(vocab=0), -1), (dict(vocab=2 ** 20 + 1, row_pitch=2 ** 21), -3), (dict(row_pitch=99), -1),
    (dict(logits=None), -2), (dict(uniforms=None), -2), (dict(tokens=None), -2),
    (dict(vocab=100000, row_pitch=100000, work=_PTR, work_bytes=1000), -4), (dict(work=_PTR + 8), -4),
])
def test_sampling_refuses(changes, code):
    args = N.SampleArgs(_PTR, 100, 0, 2, 100, _PTR, 0, None, None, None, None, 1.0, 0, 1.0, 0.0, _PTR, _PTR, None)
    assert _call("sah_sample_tokens", _changed(args, changes)) == code


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_workspaces_follow_the_work(dtype, dim):
    """What a call needs grows with its work up to a full card's, and a short one does not hold that."""
    def floats(tokens, context, requests=1):
        args = N.PagedAttentionArgs(dtype=dtype, n_requests=requests, n_tokens=tokens, Hq=8, Hkv=2, D=dim, n_pages=100, page_size=16, table_width=2 ** 14,
                                    table_pitch=2 ** 14, max_context=context)
        return N.paged_work_floats(args)

    full = floats(8192, 0)
    assert 0 < floats(1, 100) <= floats(1, 1000) <= floats(1, 10000) <= floats(16, 100000)
    assert floats(70, 70) * 10 < full and floats(1, 100) * 4 < 2 ** 20
    # a length that is not known counts as the table's, and neither more requests nor longer ones need more than a full card
    assert floats(8192, 10 ** 9) == full == floats(8192, 2 ** 18) == floats(8192, 2 ** 18, 64)


def test_nothing_to_do_is_no_error():
    lib = N.lib()
    assert lib.sah_paged_store(ctypes.byref(N.PagedStoreArgs(Hkv=1, D=8, n_pages=1, page_size=1))) == 0
    assert lib.sah_sample_tokens(ctypes.byref(N.SampleArgs(vocab=5))) == 0


def test_tensors_on_the_host_are_refused():
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 4, dtype=torch.int32)
    cache = torch.zeros(8, 16, 2, 64)
    rows = torch.zeros(3, 2, 64)
    for call in (lambda: P.assign_pages(i32, i32, table, i32, i32[:1], 16, 3),
                 lambda: P.release_pages(torch.zeros(2, dtype=torch.bool), i32, table, i32, i32[:1], 16),
                 lambda: P.store_paged(rows, rows, cache, cache, torch.zeros(3, dtype=torch.int64)),
                 lambda: P.paged_attention(rows, cache, cache, table, i32, torch.zeros(3, dtype=torch.int32), 1.0),
                 lambda: S.sample_tokens(torch.zeros(2, 10), torch.zeros(2))):
        with pytest.raises(N.NativeLibraryError, match="no CPU fallback"):
            call()


def test_a_cache_of_impossible_sizes_is_refused():
    with pytest.raises(ValueError, match="power of two"):
        P.PagedKVCache(1, 4, 24, 2, 64, 2, 100, torch.float32, "cpu")
    with pytest.raises(ValueError, match="positive"):
        P.PagedKVCache(1, 0, 16, 2, 64, 2, 100, torch.float32, "cpu")
    with pytest.raises(ValueError, match="unsupported dtype"):
        P.PagedKVCache(1, 4, 16, 2, 64, 2, 100, torch.float64, "cpu")
