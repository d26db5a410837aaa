"""A paged cache's operators against plain implementations in 64 bits: places for new tokens, stores, attention."""
import math
import random

import pytest
import torch

from sparse_attention_hub_amd.sparse_attention.utils import paged_cache as P

pytestmark = pytest.mark.gpu
_HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


# ------------------------------------------------------------------------------------------------------------ assign, release
class PlainPages:
    """The rules of include/sah_serve.h, one request after the other."""

    def __init__(self, lens, table, free, count, page):
        self.lens, self.table, self.free, self.count, self.page = list(lens), [list(r) for r in table], list(free), count, page

    def assign(self, new, n_tokens):
        slots, positions, cu, kv, granted = [-1] * n_tokens, [0] * n_tokens, [0], [], []
        row, wanted, given = 0, 0, 0
        for b, n in enumerate(new):
            n = max(n, 0)
            length = self.lens[b]
            had, has = -(-length // self.page), -(-(length + n) // self.page)
            fits = length >= 0 and row + n <= n_tokens and has <= len(self.table[b])
            need = has - had if fits else 0
            ok = fits and (need == 0 or wanted + need <= self.count)
            if ok:
                for i in range(need):
                    self.table[b][had + i] = self.free[self.count - 1 - wanted - i]
                given = max(given, wanted + need if need else 0)
                self.lens[b] += n
            for i in range(n):
                if row + i < n_tokens:
                    positions[row + i] = length + i
                    if ok:
                        slots[row + i] = self.table[b][(length + i) // self.page] * self.page + (length + i) % self.page
            wanted += need
            row += n
            cu.append(min(row, n_tokens))
            kv.append(length + n if ok else 0)
            granted.append(ok)
        self.count -= given
        return slots, positions, cu, kv, granted

    def release(self, finished):
        for b, f in enumerate(finished):
            if f:
                for j in range(-(-self.lens[b] // self.page)):
                    self.free[self.count] = self.table[b][j]
                    self.count += 1
                    self.table[b][j] = -1
                self.lens[b] = 0


def _state(lens, width, pages, page, seed):
    rng = random.Random(seed)
    order = list(range(pages))
    rng.shuffle(order)
    table = [[-1] * width for _ in lens]
    for b, n in enumerate(lens):
        for j in range(-(-n // page)):
            table[b][j] = order.pop()
    return PlainPages(lens, table, order + [-1] * (pages - len(order)), len(order), page)


def _i32(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def _on_device(plain, device):
    return (_i32(plain.lens, device), _i32(plain.table, device), _i32(plain.free, device), _i32([plain.count], device))


def _same(got, want):
    slots, positions, cu, kv, granted = want
    assert got.slot_map.tolist() == slots and got.positions.tolist() == positions
    assert got.cu_new.tolist() == cu and got.kv_lens.tolist() == kv and got.granted.tolist() == granted


@pytest.mark.parametrize("requests, page, new_hi, pad, spare", [
    (1, 16, 1, 0, 4), (1, 1, 7, 0, 50), (3, 16, 40, 5, 100), (7, 8, 1, 0, 0), (64, 16, 2, 3, 1000), (65, 32, 300, 0, 9), (257, 16, 33, 17, 100),
    (1025, 16, 12, 1, 5000), (1100, 64, 1, 0, 30), (4096, 8, 3, 0, 900), (5, 24, 2000, 100, 1000),
])
def test_assign_pages(cuda, requests, page, new_hi, pad, spare):
    """Steps on the same state, with too few pages in some; the odd page sizes are for this operator and the store alone."""
    rng = random.Random(requests + page)
    lens = [rng.choice((0, page, rng.randrange(0, 5 * page))) for _ in range(requests)]
    used = sum(-(-n // page) for n in lens)
    plain = _state(lens, 10 + -(-2 * new_hi // page), used + spare, page, requests)
    dev_lens, table, free, count = _on_device(plain, cuda)
    for step in range(3):
        new = [rng.choice((0, 1, rng.randrange(0, new_hi + 1), new_hi)) for _ in range(requests)]
        if step == 1:
            new[0] = -3
        n_tokens = max(0, sum(max(n, 0) for n in new) + pad - (2 if step == 2 else 0))  # the last step: not even rows for all
        got = P.assign_pages(_i32(new, cuda), dev_lens, table, free, count, page, n_tokens)
        _same(got, plain.assign(new, n_tokens))
        assert dev_lens.tolist() == plain.lens and count.tolist() == [plain.count] and table.tolist() == plain.table
        finished = [rng.random() < 0.3 for _ in range(requests)]
        P.release_pages(torch.tensor(finished, device=cuda), dev_lens, table, free, count, page)
        plain.release(finished)
        assert dev_lens.tolist() == plain.lens and count.tolist() == [plain.count] and table.tolist() == plain.table
        assert free.tolist()[: plain.count] == plain.free[: plain.count]


def test_assign_pages_refused_requests_and_outputs_of_their_own(cuda):
    """A full table, a corrupt length, a list that is too short: those requests get nothing, the others what they ask for."""
    page = 4
    plain = PlainPages([16, 3, -2, 4, 7, 2], [[0, 1, 2, 3], [4, -1, -1, -1], [-1] * 4, [5, -1, -1, -1], [6, 7, -1, -1], [8, -1, -1, -1]],
                       [10, 11, 12, -1], 3, page)
    lens, table, free, count = _on_device(plain, cuda)
    lens_out, count_out = torch.full_like(lens, 99), torch.full_like(count, 99)
    new = [1, 6, 1, 12, 1, 1]
    got = P.assign_pages(_i32(new, cuda), lens, table, free, count, page, 30, lens_out=lens_out, free_count_out=count_out)
    before = list(plain.lens)
    want = plain.assign(new, 30)
    _same(got, want)
    assert want[4] == [False, True, False, False, True, True]
    assert lens.tolist() == before and count.tolist() == [3] and lens_out.tolist() == plain.lens and count_out.tolist() == [1]
    wide = torch.full((6, 9), 77, dtype=torch.int32, device=cuda)  # a table that is a view of a wider one
    wide[:, :4] = table
    again = P.assign_pages(_i32([0, 1, 0, 0, 0, 1], cuda), lens_out, wide[:, :4], free, count_out, page, 2)
    _same(again, plain.assign([0, 1, 0, 0, 0, 1], 2))
    assert wide[:, 4:].eq(77).all() and wide[:, :4].tolist() == plain.table


def test_assign_pages_of_no_tokens(cuda):
    plain = _state([5, 0], 3, 6, 4, 0)
    lens, table, free, count = _on_device(plain, cuda)
    got = P.assign_pages(_i32([0, 0], cuda), lens, table, free, count, 4, 0)
    _same(got, plain.assign([0, 0], 0))
    assert lens.tolist() == [5, 0]


@pytest.mark.parametrize("requests, page, pages_each, room", [
    (1, 4, 3, 100), (1, 1, 5000, 10000), (3, 16, 2048, 10000), (7, 8, 40, 150), (300, 2, 20, 10000), (4096, 16, 3, 20000), (5, 1, 4500, 9000),
])
def test_release_pages_that_are_not_there_and_a_list_that_is_full(cuda, requests, page, pages_each, room):
    """Entries below 0 inside a request's length are no pages: they are not handed out again. Where the list is full the rest is lost; the
    requests' rows are empty all the same, and other rows as they were."""
    rng = random.Random(requests)
    width = pages_each + 2
    held = [rng.randrange(0, pages_each + 1) for _ in range(requests)]
    held[-1] = pages_each
    lens = [n * page - rng.randrange(0, page) if n else 0 for n in held]
    table = [[rng.choice((-1, -7, 5, 1000, 2 ** 31 - 1)) if rng.random() < 0.2 else rng.randrange(0, 10 ** 6) for _ in range(width)] for _ in range(requests)]
    finished = [rng.random() < 0.6 for _ in range(requests)]
    finished[-1] = True
    if requests > 2:
        lens[0], finished[0], finished[1] = -3, True, False  # a corrupt length
    free, count = [-9] * room, 2
    dev_lens, dev_table, dev_free, dev_count = _i32(lens, cuda), _i32(table, cuda), _i32(free, cuda), _i32([count], cuda)
    P.release_pages(torch.tensor(finished, device=cuda), dev_lens, dev_table, dev_free, dev_count, page)
    for b in range(requests):
        if finished[b]:
            for j in range(-(-max(lens[b], 0) // page)):
                if table[b][j] >= 0 and count < room:
                    free[count] = table[b][j]
                    count += 1
                table[b][j] = -1
            lens[b] = 0
    assert dev_count.tolist() == [count] and dev_free.tolist() == free
    assert dev_lens.tolist() == lens and dev_table.tolist() == table


# -------------------------------------------------------------------------------------------------------------------- store
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens, heads, dim, page, layout", [
    (1, 1, 8, 1, "plain"), (5, 2, 64, 16, "plain"), (300, 8, 128, 16, "heads_first"), (33, 3, 80, 8, "plain"), (17, 2, 20, 4, "plain"),
    (64, 1, 7, 3, "heads_first"), (128, 4, 64, 32, "fused"), (9, 2, 16, 16, "shifted"),
])
def test_store_paged(cuda, dtype, tokens, heads, dim, page, layout):
    pages = -(-3 * tokens // page)
    g = torch.Generator(device=cuda).manual_seed(tokens + dim)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=cuda).to(dtype)

    if layout == "heads_first":
        kc, vc = (randn(pages, heads, page, dim).transpose(1, 2) for _ in range(2))
    elif layout == "shifted":
        kc, vc = (randn(pages * page * heads * dim + 1)[1:].view(pages, page, heads, dim) for _ in range(2))
    else:
        kc, vc = (randn(2, pages, page, heads, dim).unbind(0))
    if layout == "fused":
        k, v = randn(tokens, 2 * heads, dim).split(heads, dim=1)
    else:
        k, v = randn(tokens, heads, dim), randn(tokens, heads, dim)
    slots = torch.randperm(pages * page, generator=g, device=cuda)[:tokens].clone()
    slots[::7] = -1
    slots[3::11] = pages * page + 5
    want_k, want_v = kc.clone(), vc.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want_k[s // page, s % page], want_v[s // page, s % page] = k[t], v[t]
    P.store_paged(k, v, kc, vc, slots)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_store_paged_of_no_tokens(cuda):
    c = torch.ones(2, 4, 1, 8, device=cuda)
    P.store_paged(torch.empty(0, 1, 8, device=cuda), torch.empty(0, 1, 8, device=cuda), c, c.clone(), torch.empty(0, dtype=torch.int64, device=cuda))
    assert c.eq(1).all()


# ---------------------------------------------------------------------------------------------------------------- attention
def _plain_attention(q, k, v, visible, scaling, sink):
    """One request and head in 64 bits. Returns the output and sum_j p_j |v_j|."""
    s = (q @ k.T) * scaling
    s = s.masked_fill(~visible, -math.inf)
    m = s.amax(1, keepdim=True)
    if sink is not None:
        m = m.clamp(min=sink)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(s - m)
    total = e.sum(1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - m)
    p = torch.where(total > 0, e / total, 0.0)
    return p @ v, p @ v.abs()


def _attention_case(cuda, dtype, new, cached, q_heads, kv_heads, dim, page, sink=0, window=0, sinks=False, pad=0, seed=0, layout="plain",
                    max_context=None, scale=1.0, missing=()):
    """Runs paged_attention on a cache whose every entry that belongs to no visible key is NaN, and compares."""
    g = torch.Generator().manual_seed(seed)
    kv = [a + b for a, b in zip(new, cached)]
    need = [-(-n // page) for n in kv]
    width, pages = max(max(need), 1) + 2, sum(need) + 3
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(kv), width), -1, dtype=torch.int32)
    table[:, 0] = pages + 7  # what no request holds may be anything
    kc = torch.full((pages, page, kv_heads, dim), math.nan)
    vc = torch.full((pages, page, kv_heads, dim), math.nan)
    keys = [torch.randn(n, kv_heads, dim, generator=g).to(dtype).float() for n in kv]
    values = [torch.randn(n, kv_heads, dim, generator=g).to(dtype).float() for n in kv]
    for b, n in enumerate(kv):
        for j in range(need[b]):
            at = order.pop()
            table[b, j] = at
            part = slice(j * page, min(n, (j + 1) * page))
            if (b, j) not in missing:
                kc[at, : part.stop - part.start], vc[at, : part.stop - part.start] = keys[b][part], values[b][part]
            else:
                table[b, j] = -1 if j % 2 else pages
    tokens = sum(new) + pad
    q = (scale * torch.randn(tokens, q_heads, dim, generator=g)).to(dtype)
    logit = torch.randn(q_heads, generator=g) if sinks else None
    scaling = dim ** -0.5

    def place(t):
        t = t.to(dtype)
        if layout == "heads_first":
            return t.transpose(1, 2).contiguous().to(cuda).transpose(1, 2)
        if layout == "interleaved":  # keys and values of a page beside each other
            return torch.stack([t, torch.full_like(t, math.nan)], dim=1).to(cuda)[:, 0]
        return t.to(cuda)

    queries = q.to(cuda)
    if layout == "interleaved":  # a view of a fused projection's output
        queries = torch.cat([q, torch.full_like(q, math.nan)], dim=1).to(cuda)[:, :q_heads]
    out = torch.full((tokens, q_heads, dim), 7.0, dtype=dtype, device=cuda)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    got = P.paged_attention(queries, place(kc), place(vc), table.to(cuda), _i32(kv, cuda), _i32(cu, cuda), scaling, max_context=max_context,
                            sink_size=sink, window_size=window, sinks=None if logit is None else logit.to(cuda), out=out)
    assert got is out
    got = got.double().cpu()
    assert got[cu[-1]:].eq(7).all(), "rows behind the last request's were written"
    half = _HALF_STEP[dtype]
    off2 = norm2 = most = 0.0
    for b, n in enumerate(kv):
        if not new[b]:
            continue
        position = torch.arange(cached[b], n)[:, None]
        j = torch.arange(n)[None]
        visible = j <= position
        if window:
            visible &= (j < sink) | (j > position - window)
        for miss_b, miss in missing:
            if miss_b == b:
                visible &= (j // page != miss)
        for h in range(q_heads):
            kk, vv = keys[b][:, h * kv_heads // q_heads].double(), values[b][:, h * kv_heads // q_heads].double()
            qq = q[cu[b]:cu[b + 1], h].double()
            want, size = _plain_attention(qq, kk, vv, visible, scaling, None if logit is None else float(logit[h]))
            have = got[cu[b]:cu[b + 1], h]
            # A product of D terms in fp32 is off by at most D 2^-24 sum |q k|, a logit by that and a rounding or two of its own
            # size, its weight relatively by as much (exp: a few 2^-24 more). A weight enters the second product with half a step
            # of the tensor's type, the sum of n of them is off by at most n 2^-24 (in blocks: far less), and the result is
            # rounded once.
            reach = float((qq.abs() @ kk.abs().T).max()) * scaling if n else 0.0
            logit_off = (dim + 4) * 2.0 ** -24 * reach + 8 * 2.0 ** -24
            bound = want.abs() * half + size * ((half if dtype != torch.float32 else 0.0) + 2 * logit_off + (2 * n + 16) * 2.0 ** -24) + 1e-30
            bad = (have - want).abs() > bound * 1.001
            assert not bad.any() and torch.isfinite(have).all(), (b, h, float(((have - want).abs() / bound).max()))
            most = max(most, reach)
            off2 += float((have - want).square().sum())
            norm2 += float(want.square().sum())
    # Roundings of independent signs: half a step for the weights, half for the result. A logit that is the difference of
    # partial sums of up to `most` = scale sum |q k| is rounded with 2^-24 of those at each of its last few additions (the early
    # ones are of small sums, and signs differ: 4 count), and its weight is off by as much relatively, that of the row's largest too: 8.
    # (At most = 100 that is 5e-5, where the other terms are 1e-6.)
    assert math.sqrt(off2) <= math.sqrt(norm2) * (2 * half + 2.0 ** -20 + 8 * 2.0 ** -24 * most) + 1e-30
    return got


_TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("dim", [8, 16, 40, 64, 80, 96, 128, 136, 192, 256])
def test_attention_head_dims(cuda, dtype, dim):
    _attention_case(cuda, dtype, [1, 5, 70], [130, 0, 61], 6, 2, dim, 16, seed=dim)


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("q_heads, kv_heads", [(1, 1), (8, 8), (3, 1), (8, 2), (16, 2), (32, 1), (40, 1), (132, 2)])
def test_attention_head_groups(cuda, dtype, q_heads, kv_heads):
    _attention_case(cuda, dtype, [1, 9, 0, 1], [63, 64, 200, 0], q_heads, kv_heads, 64, 8, seed=q_heads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [1, 2, 8, 32, 64, 128, 512])
def test_attention_page_sizes(cuda, dtype, page):
    _attention_case(cuda, dtype, [1, 33, 4], [600, 97, 5], 4, 1, 128, page, seed=page, layout="heads_first" if page % 3 else "interleaved")


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("cached", [0, 1, 31, 32, 33, 63, 64, 127, 128, 1000, 4097])
def test_attention_single_tokens(cuda, dtype, cached):
    _attention_case(cuda, dtype, [1] * 3, [cached, cached // 2, 0], 8, 2, 128, 16, seed=cached, pad=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("scale", [1.0, 4.0])
def test_attention_of_few_rows_is_rounded_once(cuda, dtype, dim, scale):
    """Up to 32 rows a request: weights are taken apart into two terms of the type, so that what is left is the result's own rounding."""
    page, heads, kv_heads = 16, 8, 2
    new, kv = [1, 2, 1, 8], [5000, 700, 64, 1500]
    g = torch.Generator().manual_seed(dim)
    width = -(-max(kv) // page)
    kc, vc = (torch.randn(len(kv) * width * page, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    q = (scale * torch.randn(sum(new), heads, dim, generator=g)).to(dtype)
    cu = [sum(new[:b]) for b in range(len(new) + 1)]
    table = torch.arange(len(kv) * width, dtype=torch.int32, device=cuda).view(len(kv), width)
    got = P.paged_attention(q.to(cuda), kc.to(cuda).view(-1, page, kv_heads, dim), vc.to(cuda).view(-1, page, kv_heads, dim), table, _i32(kv, cuda),
                            _i32(cu, cuda), dim ** -0.5).double().cpu()
    half = _HALF_STEP[dtype]
    for b, n in enumerate(kv):
        visible = torch.arange(n)[None] <= torch.arange(n - new[b], n)[:, None]
        at = slice(b * width * page, b * width * page + n)
        for h in range(heads):
            qq, kk, vv = q[cu[b]:cu[b + 1], h].double(), kc[at, h * kv_heads // heads].double(), vc[at, h * kv_heads // heads].double()
            want, size = _plain_attention(qq, kk, vv, visible, dim ** -0.5, None)
            # _attention_case's bound with weights off by half a step of half a step, and by what fp16's smallest number (2^-24, weights
            # above their true size by 2^3 at least) cuts off: 2^-27 of the row's largest weight, n of them
            reach = float((qq.abs() @ kk.abs().T).max()) * dim ** -0.5
            logit_off = (dim + 4) * 2.0 ** -24 * reach + 8 * 2.0 ** -24
            bound = want.abs() * half + size * (half * half + 2 * logit_off + (2 * n + 16) * 2.0 ** -24)
            if dtype == torch.float16:
                bound = bound + n * 2.0 ** -27 * float(vv.abs().max()) + 2.0 ** -25
            bad = (got[cu[b]:cu[b + 1], h] - want).abs() > bound * 1.001
            assert not bad.any(), (b, h, int(bad.sum()))


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("new, cached", [([2], [0]), ([31, 32, 33], [1, 0, 64]), ([128], [500]), ([129, 1], [0, 3000]), ([300], [17]),
                                         ([0, 0, 3], [50, 0, 0]), ([1] * 40, list(range(40)))])
def test_attention_chunks(cuda, dtype, new, cached):
    _attention_case(cuda, dtype, new, cached, 8, 2, 128, 16, seed=len(new), pad=3, layout="interleaved")


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("sink, window", [(0, 1), (0, 64), (1, 1), (4, 63), (128, 512), (100, 100000), (5000, 7)])
def test_attention_sink_and_window(cuda, dtype, sink, window):
    _attention_case(cuda, dtype, [1, 100, 1, 37], [3000, 900, 2, 0], 6, 2, 64, 16, sink=sink, window=window, seed=window)


@pytest.mark.parametrize("dtype", _TYPES)
def test_attention_sink_logits(cuda, dtype):
    _attention_case(cuda, dtype, [1, 40, 1], [2000, 10, 0], 8, 2, 64, 16, sinks=True)
    _attention_case(cuda, dtype, [1, 40, 1], [2000, 10, 0], 8, 2, 64, 16, sinks=True, sink=2, window=50)


@pytest.mark.parametrize("dtype", _TYPES)
def test_attention_pages_that_are_not_there(cuda, dtype):
    """Entries of the table outside the cache: their keys do not exist; a row that loses all of them is 0."""
    got = _attention_case(cuda, dtype, [1, 20, 3, 1], [100, 70, 0, 700], 4, 2, 64, 16, missing=((0, 2), (0, 3), (1, 4), (2, 0), (3, 0), (3, 43)))
    assert got[21:24].eq(0).all()
    _attention_case(cuda, dtype, [1, 20, 3], [100, 70, 0], 4, 2, 64, 16, sinks=True, missing=((1, 0), (2, 0)))


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("max_context", [1, 100, 5000, 10 ** 9])
def test_attention_does_not_depend_on_the_hint(cuda, dtype, max_context):
    _attention_case(cuda, dtype, [1, 50], [5000, 300], 8, 2, 128, 32, max_context=max_context)


@pytest.mark.parametrize("dtype", _TYPES)
def test_attention_of_large_logits(cuda, dtype):
    """Peaked rows: one key takes nearly all of the weight, maxima keep rising."""
    _attention_case(cuda, dtype, [1, 80], [900, 400], 4, 1, 64, 16, scale=12.0)


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("dim, window", [(64, 0), (128, 0), (128, 100), (256, 0)])
@pytest.mark.parametrize("new, cached", [
    ([1] * 30, [7 * i for i in range(30)]),                        # short tiles only
    ([1] * 20 + [0, 1], [90] * 20 + [500, 9000]),                  # ... and one long one
    ([200, 1, 1, 33, 1, 300], [0, 800, 0, 100, 5000, 50]),
    ([64] * 40, [i % 7 * 60 for i in range(40)]),
])
def test_attention_of_short_requests(cuda, dtype, dim, window, new, cached):
    """Tiles that are short enough for one workgroup, alone and beside ones that are shared."""
    _attention_case(cuda, dtype, new, cached, 8, 2, dim, 16, sink=5 if window else 0, window=window)


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("n, new", [(700, 1), (513, 0), (300, 17)])
def test_attention_of_more_requests_than_threads(cuda, dtype, n, new):
    _attention_case(cuda, dtype, [new if b % 9 else 1 - new for b in range(n)] if new < 2 else [new] * n, [b % 41 for b in range(n)], 4, 1, 64, 16)


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_values_that_are_not_finite_among_short_requests(cuda, dtype, new):
    """Only the request that holds them is changed, and of it only the rows that see them."""
    n, page, dim, heads, at = 24, 16, 64, 4, 17
    g = torch.Generator().manual_seed(9)
    kv = [new + 20 + 9 * b for b in range(n)]
    width = -(-max(kv) // page)
    kc, vc = (torch.randn(n * width, page, 1, dim, generator=g).to(dtype).to(cuda) for _ in range(2))
    table = torch.arange(n * width, dtype=torch.int32, device=cuda).view(n, width)
    q = torch.randn(n * new, heads, dim, generator=g).to(dtype).to(cuda)
    args = (table, _i32(kv, cuda), _i32([new * b for b in range(n + 1)], cuda), 0.125)
    clean = P.paged_attention(q, kc, vc, *args)
    assert bool(clean.isfinite().all())
    for b in (0, 5, 23):
        spoilt = vc.clone()
        spoilt.view(n, width * page, dim)[b, at, 3] = math.nan
        got = P.paged_attention(q, kc, spoilt, *args)
        rows = torch.arange(new * b + max(0, at - (kv[b] - new)), new * (b + 1), device=cuda)  # they see the key
        assert bool(got[rows, :, 3].isnan().all())
        same = torch.ones(n * new, dtype=torch.bool, device=cuda)
        same[new * b: new * (b + 1)] = False
        assert torch.equal(got[same], clean[same])
        before = torch.arange(new * b, int(rows[0]), device=cuda)
        assert bool(got[before].isfinite().all()) and bool(got[rows][:, :, [i for i in range(dim) if i != 3]].isfinite().all())


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_values_that_are_not_finite_stay_where_they_are_seen(cuda, dtype, bad):
    """A key or value that is not finite reaches the rows that see it and no other."""
    page, n, dim, at = 16, 70, 64, 40
    g = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn(n, 1, dim, generator=g).to(dtype) for _ in range(3))
    clean = None
    for what in ("none", "value", "key"):
        kk, vv = k.clone(), v.clone()
        if what == "value":
            vv[at, 0, 5] = bad
        if what == "key":
            kk[at] = bad
        pages = -(-n // page)
        kc, vc = torch.zeros(pages, page, 1, dim, dtype=dtype, device=cuda), torch.zeros(pages, page, 1, dim, dtype=dtype, device=cuda)
        kc.view(-1, 1, dim)[:n], vc.view(-1, 1, dim)[:n] = kk.to(cuda), vv.to(cuda)
        out = P.paged_attention(q.to(cuda), kc, vc, torch.arange(pages, dtype=torch.int32, device=cuda)[None], _i32([n], cuda), _i32([0, n], cuda),
                                dim ** -0.5).float().cpu()
        if what == "none":
            clean = out
            continue
        # rows before the bad key: the same up to the roundings of another order of sums (each side off by two half steps)
        assert torch.allclose(out[:at], clean[:at], rtol=0, atol=8 * _HALF_STEP[dtype] * float(v.abs().max()))
        if what == "value":
            others = torch.arange(dim) != 5
            if bad != bad:
                assert out[at:, 0, 5].isnan().all()
            else:
                assert out[at:, 0, 5].eq(bad).all()
            assert torch.allclose(out[at:, 0][:, others], clean[at:, 0][:, others], rtol=0, atol=8 * _HALF_STEP[dtype] * float(v.abs().max()))
        else:
            # q . k is NaN (infinities of both signs, or NaN itself), and so is the row
            assert out[at:].isnan().all()


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new, kv_heads", [(1, 1), (1, 2), (4, 2), (9, 1)])
def test_values_that_are_not_finite_in_a_long_context(cuda, dtype, dim, new, kv_heads):
    """Tiles of three dozen parts: a bad value spoils its own dim of the rows that see it, a bad key all of those rows, nothing else."""
    page, n, group, bad_dim = 16, 9001, 4, 3
    g = torch.Generator().manual_seed(dim + new)
    k, v = (torch.randn(n, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    q = (4 * torch.randn(new, group * kv_heads, dim, generator=g)).to(dtype)  # few keys take most of a row's weight
    pages = -(-n // page)
    table, kv, cu = torch.arange(pages, dtype=torch.int32, device=cuda)[None], _i32([n], cuda), _i32([0, new], cuda)

    def attend(keys, values):
        kc, vc = (torch.zeros(pages * page, kv_heads, dim, dtype=dtype, device=cuda) for _ in range(2))
        kc[:n], vc[:n] = keys.to(cuda), values.to(cuda)
        return P.paged_attention(q.to(cuda), kc.view(pages, page, kv_heads, dim), vc.view(pages, page, kv_heads, dim), table, kv, cu,
                                 dim ** -0.5).double().cpu()

    clean = attend(k, v)
    want, bound = torch.empty(new, group, dim, dtype=torch.float64), torch.empty(new, group, dim, dtype=torch.float64)
    visible = torch.arange(n)[None] <= torch.arange(n - new, n)[:, None]
    half = _HALF_STEP[dtype]
    for h in range(group):
        qq, kk = q[:, h].double(), k[:, 0].double()
        want[:, h], size = _plain_attention(qq, kk, v[:, 0].double(), visible, dim ** -0.5, None)
        # the bound of _attention_case
        reach = float((qq.abs() @ kk.abs().T).max()) * dim ** -0.5
        logit_off = (dim + 4) * 2.0 ** -24 * reach + 8 * 2.0 ** -24
        bound[:, h] = want[:, h].abs() * half + size * ((half if dtype != torch.float32 else 0.0) + 2 * logit_off + (2 * n + 16) * 2.0 ** -24)
    others = [d for d in range(dim) if d != bad_dim]
    for at in (0, n // 2, n - 1):
        sees = torch.arange(n - new, n) >= at
        for bad in (math.nan, math.inf):
            spoilt = v.clone()
            spoilt[at, 0, bad_dim] = bad
            got = attend(k, spoilt)
            assert torch.equal(got[:, group:], clean[:, group:])  # the other key heads
            assert got[sees, :group, bad_dim].isnan().all() if bad != bad else not got[sees, :group, bad_dim].isfinite().any()
            off = (got[:, :group] - want).abs() <= 1.001 * bound
            assert bool(off[:, :, others].all()) and bool(off[~sees].all()), (at, bad)
        spoilt = k.clone()
        spoilt[at, 0, bad_dim] = math.nan
        got = attend(spoilt, v)
        assert got[sees, :group].isnan().all() and torch.equal(got[:, group:], clean[:, group:])
        assert bool(((got[:, :group] - want).abs() <= 1.001 * bound)[~sees].all())


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("new, n", [(1, 600), (40, 600), (2, 9001), (150, 3000)])
def test_averages_of_the_largest_values_are_finite(cuda, dtype, new, n):
    """Values of the type's largest number: a weight that is rounded up, or a sum before it is divided, must not take a result past it."""
    page, dim, heads = 16, 64, 4
    most = torch.finfo(dtype).max if dtype != torch.float32 else 2.0 ** 127 * 1.9  # (fp32: its roundings' worth below the end)
    logits = torch.linspace(0.01, 3.9, new * heads)[torch.randperm(new * heads, generator=torch.Generator().manual_seed(new))]
    q = torch.zeros(new * heads, dim)
    q[:, 0] = logits
    q = q.view(new, heads, dim).to(dtype)
    pages = -(-n // page)
    kc = torch.zeros(pages * page, 1, dim)
    kc[64:, 0, 0] = 1.0  # all keys but the first ones weigh the same, a row's own number of times more than those
    signs = torch.where(torch.rand(pages * page, 1, dim, generator=torch.Generator().manual_seed(1)) < 0.5, -1.0, 1.0)
    visible = torch.arange(n)[None] <= torch.arange(n - new, n)[:, None]
    args = (torch.arange(pages, dtype=torch.int32, device=cuda)[None], _i32([n], cuda), _i32([0, new], cuda), 1.0)
    half = _HALF_STEP[dtype]
    for sign in (torch.ones_like(signs), signs):
        vc = (sign * most).to(dtype)
        got = P.paged_attention(q.to(cuda), kc.to(dtype).to(cuda).view(pages, page, 1, dim), vc.to(cuda).view(pages, page, 1, dim), *args).double().cpu()
        for h in range(heads):
            want, size = _plain_attention(q[:, h].double(), kc[:n, 0].double(), vc[:n, 0].double(), visible, 1.0, None)
            # logits are exact; weights and sums as in _attention_case
            bound = want.abs() * half + size * ((half if dtype != torch.float32 else 0.0) + (2 * n + 32) * 2.0 ** -24)
            assert bool(((got[:, h] - want).abs() <= 1.001 * bound).all()), (h, float(got[:, h].abs().max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new, n", [(1, 700), (40, 700), (1, 9001)])
def test_logits_far_below_zero_are_logits(cuda, dtype, new, n):
    """Every logit is one and the same number of -1e36 to -1e38: a row is the average of what it sees."""
    page, dim, heads = 16, 64, 4
    g = torch.Generator().manual_seed(n)
    pages = -(-n // page)
    q, kc = torch.zeros(new, heads, dim), torch.zeros(pages * page, 1, dim)
    q[:, :, 0] = torch.tensor([2.0 ** 60, 2.0 ** 61, 2.0 ** 63, 2.0 ** 66])
    kc[:, :, 0] = -2.0 ** 60
    vc = torch.randn(pages * page, 1, dim, generator=g).to(dtype)
    got = P.paged_attention(q.to(dtype).to(cuda), kc.to(dtype).to(cuda).view(pages, page, 1, dim), vc.to(cuda).view(pages, page, 1, dim),
                            torch.arange(pages, dtype=torch.int32, device=cuda)[None], _i32([n], cuda), _i32([0, new], cuda), 1.0).double().cpu()
    visible = torch.arange(n)[None] <= torch.arange(n - new, n)[:, None]
    want, size = _plain_attention(torch.zeros(new, dim).double(), torch.zeros(n, dim).double(), vc[:n, 0].double(), visible, 1.0, None)
    half = _HALF_STEP[dtype]
    # equal weights are exact; sums of n of them, and the result's rounding
    bound = want.abs() * half + size * (2 * n + 16) * 2.0 ** -24
    assert bool(((got - want[:, None]).abs() <= 1.001 * bound[:, None]).all())


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("page", [1, 64])
def test_strides_of_dimensions_of_one_entry_are_nothing(cuda, dtype, page):
    """One token, one page, one key head: their strides may be any number, as views of such tensors have them."""
    dim, heads, n = 64, 4, page
    g = torch.Generator(device=cuda).manual_seed(page)
    k, v, q = (torch.randn(m, h, dim, generator=g, device=cuda).to(dtype) for m, h in ((n, 1), (n, 1), (1, heads)))
    q = q.as_strided((1, heads, dim), (heads * dim + 3, dim, 1))
    caches = [torch.zeros(page * dim, dtype=dtype, device=cuda).as_strided((1, page, 1, dim), (7, dim if page > 1 else 5, 3, 1)) for _ in range(2)]
    for t in range(n):
        one = (x[t:t + 1].as_strided((1, 1, dim), (1, 1, 1)) for x in (k, v))
        P.store_paged(*one, *caches, torch.tensor([t], device=cuda))
    assert torch.equal(caches[0].reshape(n, dim), k[:, 0]) and torch.equal(caches[1].reshape(n, dim), v[:, 0])
    table, kv, cu = _i32([0, 7, 7], cuda).as_strided((1, 1), (3, 2)), _i32([n], cuda), _i32([0, 1], cuda)
    out = torch.empty(heads * dim, dtype=dtype, device=cuda).as_strided((1, heads, dim), (9, dim, 1))
    P.paged_attention(q, *caches, table, kv, cu, 0.125, out=out)
    want = P.paged_attention(q.contiguous(), k[None].contiguous(), v[None].contiguous(), table, kv, cu, 0.125)
    assert torch.equal(out, want)


def test_attention_offsets_beyond_32_bits(cuda):
    """Pages whose elements start past 2^31."""
    page, heads, dim, pages = 16, 8, 128, 2 ** 31 // (16 * 8 * 128) + 40
    kc = torch.empty(pages, page, heads, dim, dtype=torch.bfloat16, device=cuda)
    vc = torch.empty_like(kc)
    n = 100
    g = torch.Generator(device=cuda).manual_seed(1)
    k, v, q = (torch.randn(n, heads, dim, generator=g, device=cuda).to(torch.bfloat16) for _ in range(3))
    held = torch.tensor([pages - 1, 3, pages - 5, pages - 2, 9, pages - 30, pages - 31], dtype=torch.int32, device=cuda)
    slots = (held.long()[:, None] * page + torch.arange(page, device=cuda)).reshape(-1)[:n].contiguous()
    P.store_paged(k, v, kc, vc, slots)
    far = P.paged_attention(q, kc, vc, held[None].contiguous(), _i32([n], cuda), _i32([0, n], cuda), dim ** -0.5)
    near_k, near_v = kc[held.long()].clone(), vc[held.long()].clone()
    near = P.paged_attention(q, near_k, near_v, torch.arange(7, dtype=torch.int32, device=cuda)[None], _i32([n], cuda), _i32([0, n], cuda), dim ** -0.5)
    assert torch.equal(far, near)
    assert torch.equal(near_k.view(-1, heads, dim)[:n], k) and torch.equal(near_v.view(-1, heads, dim)[:n], v)


def test_attention_of_lengths_that_do_not_fit_is_bounded(cuda):
    """Corrupt lengths: longer than the table, shorter than the new tokens, running sums that fall or pass the rows. Nothing outside
    the tensors is touched; rows before a request's beginning see nothing."""
    dim, page = 64, 16
    kc = torch.randn(8, page, 1, dim, device=cuda).to(torch.bfloat16)
    vc = torch.randn(8, page, 1, dim, device=cuda).to(torch.bfloat16)
    table = torch.arange(8, dtype=torch.int32, device=cuda).view(2, 4).contiguous()
    q = torch.randn(6, 2, dim, device=cuda).to(torch.bfloat16)
    out = P.paged_attention(q, kc, vc, table, _i32([1000, 2], cuda), _i32([0, 2, 6], cuda), 0.125).float().cpu()
    full = P.paged_attention(q[:2], kc, vc, table[:1], _i32([64], cuda), _i32([0, 1], cuda), 0.125).float().cpu()
    assert torch.equal(out[0], full[0])          # sees all 64 keys that the table can hold
    assert out[2:4].eq(0).all() and torch.isfinite(out).all()
    for kv, cu in (([5, 5], [0, 4, 2]), ([5, 5], [0, 100, 200]), ([-4, 3], [0, 2, 4]), ([3, 3], [-5, 2, 4]), ([2 ** 31 - 1, 1], [0, 3, 6])):
        out = P.paged_attention(q, kc, vc, table, _i32(kv, cuda), _i32(cu, cuda), 0.125, out=torch.zeros_like(q))
        assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("sink, window", [(0, 0), (4, 950), (4, 920), (0, 937), (4, 900), (0, 100), (64, 1), (1, 2000)])
def test_windows_of_lengths_beyond_the_table(cuda, dtype, sink, window):
    """Positions go by the length, keys end with the table: a window may see a few of them, or the sinks alone, or nothing."""
    page, held, length, new, heads, dim = 16, 64, 1000, 3, 4, 64
    g = torch.Generator().manual_seed(window)
    q, k, v = (torch.randn(m, h, dim, generator=g).to(dtype) for m, h in ((new, heads), (held, 1), (held, 1)))
    got = P.paged_attention(q.to(cuda), k.view(-1, page, 1, dim).to(cuda), v.view(-1, page, 1, dim).to(cuda),
                            torch.arange(held // page, dtype=torch.int32, device=cuda)[None], _i32([length], cuda), _i32([0, new], cuda), 0.125,
                            sink_size=sink if window else 0, window_size=window).double().cpu()
    position, j = torch.arange(length - new, length)[:, None], torch.arange(held)[None]
    visible = ((j < sink) | (j > position - window)) if window else torch.ones(new, held, dtype=torch.bool)
    half = _HALF_STEP[dtype]
    for h in range(heads):
        want, size = _plain_attention(q[:, h].double(), k[:, 0].double(), v[:, 0].double(), visible, 0.125, None)
        bound = want.abs() * half + size * (half + 2.0 ** -16)  # (fp32 terms of _attention_case: less than the last)
        assert bool(((got[:, h] - want).abs() <= bound).all())
        assert bool(got[:, h][~visible.any(1)].eq(0).all())


# ------------------------------------------------------------------------------------------------- refusals on the device
def test_tensors_that_do_not_fit_together_are_refused(cuda):
    i32 = torch.zeros(2, dtype=torch.int32, device=cuda)
    table = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    one = i32[:1]
    for bad, match in ((dict(new_lens=i32.long()), "int32"), (dict(lens=i32[:1]), "shape"), (dict(block_table=table[:1]), "block_table"),
                       (dict(block_table=table.long()), "block_table"), (dict(free_count=i32), "free_count"), (dict(page_size=0), "page_size"),
                       (dict(n_tokens=-1), "n_tokens"), (dict(block_table=table.t()[:2]), "block_table"), (dict(lens=i32.cpu()), "expected"),
                       (dict(new_lens=i32[:0]), "at least one")):
        args = dict(dict(new_lens=i32, lens=i32, block_table=table, free_pages=i32, free_count=one, page_size=16, n_tokens=3), **bad)
        with pytest.raises(ValueError, match=match):
            P.assign_pages(**args)
    cache = torch.zeros(8, 16, 2, 64, device=cuda)
    rows, slots = torch.zeros(3, 2, 64, device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)
    for bad in (dict(keys=rows[:, :1]), dict(values=rows[:2]), dict(slot_map=slots.int()), dict(keys=rows.half()), dict(value_cache=cache[:4]),
                dict(slot_map=slots[:2]), dict(key_cache=cache.transpose(2, 3))):
        args = dict(dict(keys=rows, values=rows, key_cache=cache, value_cache=cache, slot_map=slots), **bad)
        with pytest.raises(ValueError):
            P.store_paged(**args)
    q, cu = torch.zeros(3, 4, 64, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    good = dict(queries=q, key_cache=cache, value_cache=cache, block_table=table, kv_lens=i32, cu_new=cu, scaling=1.0)
    for bad in (dict(queries=q[:, :3]), dict(queries=q.half()), dict(cu_new=i32), dict(kv_lens=i32.long()), dict(sink_size=4),
                dict(sink_size=-1, window_size=3), dict(sinks=torch.zeros(2, device=cuda)), dict(out=q[:2]), dict(max_context=-1),
                dict(scaling=math.nan), dict(queries=torch.zeros(3 * 4 * 64 + 1, device=cuda)[1:].view(3, 4, 64))):
        with pytest.raises(ValueError):
            P.paged_attention(**dict(good, **bad))


@pytest.mark.parametrize("page_size", [0, -16, 2 ** 31, 2 ** 32 + 16])
def test_page_sizes_that_do_not_fit_are_refused(cuda, page_size):
    i32, table, free = (torch.zeros(s, dtype=torch.int32, device=cuda) for s in (2, (2, 4), 8))
    with pytest.raises(ValueError, match="page_size"):
        P.assign_pages(i32, i32, table, free, i32[:1], page_size, 3)
    with pytest.raises(ValueError, match="page_size"):
        P.release_pages(torch.ones(2, dtype=torch.bool, device=cuda), i32, table, free, i32[:1], page_size)
    assert not any(t.any() for t in (i32, table, free))


@pytest.mark.parametrize("layout", ["beside", "interleaved", "heads_first", "same", "shifted", "cache"])
def test_output_and_queries_of_one_buffer(cuda, layout):
    """Slices that share nothing are what they are apart; what shares memory is refused."""
    tokens, heads, dim, page, n = 5, 4, 64, 16, 90
    g = torch.Generator(device=cuda).manual_seed(2)
    kc, vc = (torch.randn(6, page, heads, dim, generator=g, device=cuda) for _ in range(2))
    q = torch.randn(tokens, heads, dim, generator=g, device=cuda)
    args = (kc, vc, torch.arange(6, dtype=torch.int32, device=cuda)[None], _i32([n], cuda), _i32([0, tokens], cuda), 0.125)
    want = P.paged_attention(q, *args)
    if layout == "beside":
        queries, out = torch.zeros(tokens, 3 * heads, dim, device=cuda).split([heads, 2 * heads], dim=1)
        out = out[:, heads:]
    elif layout == "interleaved":
        queries, out = torch.zeros(tokens, heads, 2 * dim, device=cuda).split(dim, dim=2)
    elif layout == "heads_first":
        queries, out = torch.zeros(2 * heads, tokens, dim, device=cuda).transpose(0, 1).split(heads, dim=1)
    elif layout == "same":
        queries = out = q.clone()
    elif layout == "shifted":
        both = torch.zeros(tokens + 1, heads, dim, device=cuda)
        queries, out = both[:tokens], both[1:]
    else:
        queries, out = q.clone(), kc[0, :tokens]
    queries.copy_(q)
    if layout in ("same", "shifted", "cache"):
        with pytest.raises(ValueError, match="sah_paged_attention: out"):
            P.paged_attention(queries, *args, out=out)
        return
    assert P.paged_attention(queries, *args, out=out) is out
    assert torch.equal(out, want) and torch.equal(queries, q)


# ------------------------------------------------------------------------------------------------------ as they are used
def _dense_reference(q, k, v, scaling):
    """One request in 64 bits: the last len(q) positions' attention over all keys; (n, heads, dim) each."""
    group = q.shape[1] // k.shape[1]
    n, m = q.shape[0], k.shape[0]
    visible = torch.arange(m)[None] <= torch.arange(m - n, m)[:, None]
    out = torch.empty(q.shape, dtype=torch.float64)
    for h in range(q.shape[1]):
        out[:, h] = _plain_attention(q[:, h].double(), k[:, h // group].double(), v[:, h // group].double(), visible, scaling, None)[0]
    return out


def test_requests_that_come_and_go(cuda):
    """A cache of two layers: prompts in chunks, answers, requests that end and others that take their place."""
    dtype, dim, heads, kv_heads, page, requests = torch.bfloat16, 64, 4, 2, 16, 5
    cache = P.PagedKVCache(2, 60, page, kv_heads, dim, requests, 300, dtype, cuda)
    cache.key_cache.fill_(math.nan)
    cache.value_cache.fill_(math.nan)
    g = torch.Generator().manual_seed(0)
    rng = random.Random(0)
    history = [[None, None] for _ in range(requests)]  # (keys, values) of each layer
    for step in range(12):
        new = [rng.choice((0, 1, 1, rng.randrange(1, 60))) for _ in range(requests)]
        tokens = sum(new) + 2
        given = cache.assign(_i32(new, cuda), tokens)
        granted, cu = given.granted.tolist(), given.cu_new.tolist()
        for layer in range(2):
            q, k, v = (torch.randn(tokens, h, dim, generator=g).to(dtype) for h in (heads, kv_heads, kv_heads))
            out = cache.attend(layer, q.to(cuda), k.to(cuda), v.to(cuda), given, dim ** -0.5).double().cpu()
            for b in range(requests):
                rows = slice(cu[b], cu[b + 1])
                if not granted[b]:
                    assert out[rows].eq(0).all()
                    continue
                old = history[b][layer]
                history[b][layer] = (k[rows], v[rows]) if old is None else (torch.cat([old[0], k[rows]]), torch.cat([old[1], v[rows]]))
                if new[b]:
                    want = _dense_reference(q[rows], *history[b][layer], dim ** -0.5)
                    # 2^-8 of the weights' rounding and as much of the result's, of values up to 1 after the average
                    assert float((out[rows] - want).norm() / want.norm()) < 2 * 2.0 ** -8
        if step % 3 == 2:
            finished = [rng.random() < 0.5 for _ in range(requests)]
            cache.release(torch.tensor(finished, device=cuda))
            for b, f in enumerate(finished):
                if f:
                    history[b] = [None, None]
    assert cache.lens.tolist() == [0 if h[0] is None else len(h[0][0]) for h in history]
    held = sum(-(-n // page) for n in cache.lens.tolist())
    free = cache.free_pages[: int(cache.free_count)].tolist()
    in_use = [p for row in cache.block_table.tolist() for p in row if p >= 0]
    assert len(in_use) == held and sorted(free + in_use) == list(range(60))


def _answer_step(cache, new, q, k, v):
    given = cache.assign(new, q.shape[0])
    return cache.attend(0, q, k, v, given, 0.125, max_context=200)


def test_a_captured_step_grows_the_cache_on_every_replay(cuda):
    dim, requests = 64, 3
    g = torch.Generator(device=cuda).manual_seed(5)

    def randn(h):
        return torch.randn(requests, h, dim, generator=g, device=cuda).to(torch.float16)

    caches = [P.PagedKVCache(1, 40, 16, 2, dim, requests, 200, torch.float16, cuda) for _ in range(2)]
    prompt = _i32([5, 100, 31], cuda)
    pk, pv, pq = (torch.randn(136, h, dim, generator=g, device=cuda).to(torch.float16) for h in (2, 2, 4))
    for c in caches:
        c.attend(0, pq, pk, pv, c.assign(prompt, 136), 0.125)
    new = torch.ones(requests, dtype=torch.int32, device=cuda)
    q, k, v = randn(4), randn(2), randn(2)
    warm = P.PagedKVCache(1, 40, 16, 2, dim, requests, 200, torch.float16, cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _answer_step(warm, new, q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _answer_step(caches[0], new, q, k, v)
    for _ in range(20):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=cuda))
        graph.replay()
        want = _answer_step(caches[1], new, q, k, v)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(caches[0].lens, caches[1].lens) and caches[0].lens.tolist() == [25, 120, 51]


def test_two_streams_at_once(cuda):
    """Calls that overlap on two streams do not share anything."""
    dim = 128
    g = torch.Generator(device=cuda).manual_seed(9)
    kc, vc = (torch.randn(600, 16, 2, dim, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    table = torch.randperm(600, generator=g, device=cuda)[:500].to(torch.int32).view(2, 250)
    kv, cu = _i32([4000, 3500], cuda), _i32([0, 1, 2], cuda)
    qs = [torch.randn(2, 8, dim, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2)]
    want = [P.paged_attention(q, kc, vc, table, kv, cu, 0.1) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(P.paged_attention(qs[i], kc, vc, table, kv, cu, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
