"""sample_tokens against the rules of include/sah_serve.h in 64 bits, row by row."""
import math

import numpy as np
import pytest
import torch

from sparse_attention_hub_amd import _native as N
from sparse_attention_hub_amd.sparse_attention.utils.token_sampling import sample_tokens

pytestmark = pytest.mark.gpu
_TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _f32(v):
    return float(np.float32(v))


def _plain(x, u, t, k, p, least):
    """(token, log of its share) of one row; x float64."""
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return -1, -math.inf
    if not t > 0:
        return int(np.argmax(x)), 0.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == np.inf, 1.0, 0.0) if x.max() == np.inf else np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / t))
        if t == math.inf and x.max() < np.inf:
            w = np.where(x == -np.inf, 0.0, 1.0)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if k > 0:
        order = order[:k]
    if p < 1:
        ahead = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
        order = order[: max(1, int((ahead < p * w[order].sum()).sum()))]
    if least > 0:
        order = order[w[order] >= min(least, 1.0)]
    order = np.sort(order)
    mass = np.cumsum(w[order])
    u = 0.0 if not u > 0 else u
    at = int(np.searchsorted(mass, u * mass[-1], side="right"))
    if at >= len(order) or u >= 1:
        at = int(np.nonzero(w[order] > 0)[0][-1])
    return int(order[at]), math.log(w[order[at]] / mass[-1])


def _compare(cuda, x, u, t=None, k=None, p=None, least=None):
    """Settings: None, numbers, or lists of one value per row."""
    rows = x.shape[0]

    def given(v, dtype):
        return torch.tensor(v, dtype=dtype, device=cuda) if isinstance(v, list) else v

    tokens, logs = sample_tokens(x.to(cuda), u.to(cuda), given(t, torch.float32), given(k, torch.int32), given(p, torch.float32),
                                 given(least, torch.float32))
    assert tokens.dtype == torch.int64 and logs.dtype == torch.float32 and tokens.shape == logs.shape == (rows,)

    def each(v, off):
        return [_f32(a) for a in v] if isinstance(v, list) else [_f32(off if v is None else v)] * rows

    wide = x.double().numpy()
    for r, (tt, kk, pp, ll) in enumerate(zip(each(t, 1.0), each(k, 0), each(p, 1.0), each(least, 0.0))):
        want, log = _plain(wide[r], float(u[r]), tt, int(kk), pp, ll)
        assert int(tokens[r]) == want, (r, int(tokens[r]), want, tt, kk, pp, ll, float(u[r]))
        # the logarithm in 64 bits, rounded once to 32; sums in steps of 2^-43 add less than 2^-22
        assert float(logs[r]) == log or abs(float(logs[r]) - log) <= 2.0 ** -24 * abs(log) + 2.0 ** -22, (r, float(logs[r]), log)


def _logits(rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g)
    x[:, torch.randint(0, vocab, (3,), generator=g)] += 4.0
    return x.to(dtype), torch.rand(rows, generator=g)


_SETTINGS = [dict(), dict(t=0.7), dict(k=1), dict(k=40, t=1.3), dict(p=0.9), dict(p=0.3, t=0.5), dict(least=0.05), dict(k=50, p=0.8, least=0.02),
             dict(p=0.999, t=2.0), dict(t=0.0), dict(k=10 ** 6), dict(p=0.0), dict(least=1.0), dict(p=0.95, least=0.5, k=3)]


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("settings", _SETTINGS, ids=[str(s) for s in _SETTINGS])
def test_settings(cuda, dtype, settings):
    x, u = _logits(24, 5003, dtype, 1)
    _compare(cuda, x, u, **settings)


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 511, 1000, 1024, 1025, 4096, 8191, 8193, 32000, 65537, 131071, 262145])
def test_sizes(cuda, dtype, vocab):
    x, u = _logits(5, vocab, dtype, vocab)
    _compare(cuda, x, u, k=[0, 20, 0, 3, 0], p=[1.0, 0.9, 0.8, 1.0, 0.97], least=[0.0, 0.0, 0.1, 0.0, 0.001], t=[1.0, 0.8, 1.2, 0.0, 1.0])


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("pitch", [1000, 1001, 1003, 1024, 4099])
def test_rows_apart_and_anywhere(cuda, dtype, pitch):
    """Rows that start at any element."""
    x, u = _logits(7, 1000, dtype, pitch)
    wide = torch.full((7 * pitch + 3,), 30.0, dtype=dtype)
    view = wide[3:].as_strided((7, 1000), (pitch, 1), 3)
    view.copy_(x)
    dev = wide.to(cuda).as_strided((7, 1000), (pitch, 1), 3)
    for settings in (dict(), dict(top_p=0.9), dict(top_k=17)):
        a, b = sample_tokens(x.to(cuda), u.to(cuda), **settings), sample_tokens(dev, u.to(cuda), **settings)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    _compare(cuda, x, u, p=0.9)


@pytest.mark.parametrize("dtype", _TYPES)
def test_equal_logits(cuda, dtype):
    """Ties go to the lower index: at the largest logit, at top-k's border, at top-p's."""
    x = torch.zeros(12, 3000)
    x[:, 1000:1010] = 2.0
    x[6:, 5] = 2.0
    x[:, 2000:] = -1.0
    x[3, ::2] = -0.0
    u = torch.linspace(0, 0.9999, 12)
    for settings in (dict(), dict(t=0.0), dict(k=4), dict(k=500), dict(p=0.003), dict(p=0.4), dict(p=0.5, k=1234), dict(k=11), dict(k=12, least=0.5)):
        _compare(cuda, x.to(dtype), u, **settings)
    same = torch.full((4, 777), 1.5).to(dtype)
    for settings in (dict(k=10), dict(p=0.25), dict(p=0.25, k=100), dict(t=0.0), dict(least=1.0)):
        _compare(cuda, same, torch.tensor([0.0, 0.3, 0.77, 0.999]), **settings)


@pytest.mark.parametrize("dtype", _TYPES)
def test_logits_that_are_not_finite(cuda, dtype):
    x, u = _logits(10, 2500, dtype, 3)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 1::2] = -math.inf
    x[3, 40:] = math.nan
    x[4, [7, 900, 901]] = math.inf
    x[5] = math.inf
    x[6] = -math.inf
    x[6, 2499] = -3.0
    x[7, 0] = math.inf
    x[8] = torch.finfo(dtype).min
    x[9] = torch.finfo(dtype).min
    x[9, 77] = torch.finfo(dtype).max
    for settings in (dict(), dict(t=0.0), dict(k=5), dict(p=0.9), dict(least=0.1), dict(k=2000, p=0.99, t=0.5)):
        _compare(cuda, x, u, **settings)


@pytest.mark.parametrize("dtype", _TYPES)
def test_random_numbers_and_settings_at_their_ends(cuda, dtype):
    x, _ = _logits(9, 999, dtype, 4)
    u = torch.tensor([0.0, 2.0 ** -24, 1 - 2.0 ** -24, 1.0, 5.0, -1.0, math.nan, 0.5, 1 - 2.0 ** -53], dtype=torch.float64)
    for v in (u, u.float()):
        for settings in (dict(), dict(k=3), dict(p=0.5)):
            _compare(cuda, x, v, **settings)
    _compare(cuda, x, u, t=[0.0, -1.0, math.nan, math.inf, 1e-6, 1e6, 1e-30, 1.0, 100.0])
    _compare(cuda, x, u, k=[0, -5, 1, 2, 998, 999, 1000, 2 ** 31 - 1, -2 ** 31])
    _compare(cuda, x, u, p=[0.0, -1.0, 1.0, 2.0, 1e-9, 1 - 2.0 ** -24, 0.5, math.inf, 1e-30])
    _compare(cuda, x, u, least=[0.0, -1.0, 1.0, 7.0, 1e-9, 0.999, 0.5, 1e-30, math.inf])
    _compare(cuda, x, u, p=[math.nan] * 9, least=[math.nan] * 9)


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("spread", [0.0001, 0.05, 0.7, 30.0, 3000.0])
def test_narrow_and_wide_rows(cuda, dtype, spread):
    """Logits that lie close together or far apart, around a large offset too: thresholds among many nearly equal values."""
    x, u = _logits(8, 20011, dtype, 11, spread)
    for y in (x, (x.float() + 100.0).to(dtype), (x.float() * 1e-3 - 50.0).to(dtype)):
        for settings in (dict(), dict(k=1000), dict(p=0.6), dict(k=9000, p=0.7), dict(k=19000, p=0.99, least=1e-4)):
            _compare(cuda, y, u, **settings)


def test_more_rows_than_the_chip_holds_at_once(cuda):
    x, u = _logits(700, 3001, torch.bfloat16, 21)
    _compare(cuda, x, u, t=0.9, p=0.95)


@pytest.mark.parametrize("vocab", [8193, 9000, 20000])
@pytest.mark.parametrize("settings", [dict(top_p=0.9), dict(top_p=0.97, temperature=1.4), dict(top_p=0.9, min_p=0.01)])
def test_selections_that_follow_each_other_at_once(cuda, vocab, settings):
    """Rows just longer than the list, where a wave's pass between the list's threshold and the nucleus' border is a few loads: every run the same."""
    x, u = _logits(1000, vocab, torch.float32, vocab)
    x[::2] = x[::2].to(torch.bfloat16).float()
    few = slice(0, 1000, 50)
    _compare(cuda, x[few].contiguous(), u[few].contiguous(), t=settings.get("temperature"), p=settings["top_p"], least=settings.get("min_p"))
    x, u = x.to(cuda), u.to(cuda)
    tokens, logs = sample_tokens(x, u, **settings)
    for _ in range(20):
        again, again_logs = sample_tokens(x, u, **settings)
        assert torch.equal(again, tokens) and torch.equal(again_logs, logs)


def test_no_rows(cuda):
    tokens, logs = sample_tokens(torch.empty(0, 100, device=cuda), torch.empty(0, device=cuda))
    assert tokens.shape == (0,) and logs.shape == (0,)


def test_the_same_numbers_give_the_same_tokens_in_a_replayed_graph(cuda):
    x, u = (t.to(cuda) for t in _logits(33, 50001, torch.float32, 8))
    settings = dict(temperature=0.8, top_p=0.9, top_k=torch.arange(33, dtype=torch.int32, device=cuda) * 7, min_p=0.01)
    sample_tokens(x, u, **settings)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, logs = sample_tokens(x, u, **settings)
    for seed in range(4):
        new_x, new_u = _logits(33, 50001, torch.float32, 30 + seed)
        x.copy_(new_x)
        u.copy_(new_u)
        graph.replay()
        want = sample_tokens(x, u, **settings)
        torch.cuda.synchronize()
        assert torch.equal(tokens, want[0]) and torch.equal(logs, want[1])


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("rows, vocab", [(1, 65535), (1, 65536), (2, 65537), (3, 65536 + 2049), (17, 70001), (64, 100001), (128, 66001), (129, 66001)])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=1000), dict(top_k=3, top_p=0.5), dict(top_p=0.9), dict(top_p=0.999, temperature=2.0), dict(min_p=0.1),
                                      dict(top_k=5000)])
def test_several_workgroups_a_row_or_one(cuda, dtype, rows, vocab, settings):
    """The results of rows shared by several workgroups are those of one workgroup each, also where a part of the row is hidden."""
    x, u = _logits(rows, vocab, dtype, 5)
    x, u = x.to(cuda), u.to(cuda)
    x[0, : vocab // 2] = -math.inf
    x[rows // 2, 1000:] = -math.inf
    tokens, logs = sample_tokens(x, u, **settings)
    one, one_log = torch.empty_like(tokens), torch.empty_like(logs)
    full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings)
    args = N.SampleArgs(x.data_ptr(), vocab, N.dtype_code(dtype), rows, vocab, u.data_ptr(), int(u.dtype == torch.float64), None, None, None, None,
                        full["temperature"], full["top_k"], full["top_p"], full["min_p"], one.data_ptr(), one_log.data_ptr(), N.stream_ptr(x.device))
    N.call_on(x.device, "sah_sample_tokens", args)
    assert torch.equal(tokens, one) and torch.equal(logs, one_log)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=20), dict(top_p=0.95, temperature=1.3)])
def test_rows_shared_by_workgroups_in_a_replayed_graph_and_on_two_streams(cuda, settings):
    rows, vocab = 3, 70001
    x, u = (t.to(cuda) for t in _logits(rows, vocab, torch.bfloat16, 40))
    sample_tokens(x, u, **settings)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, logs = sample_tokens(x, u, **settings)
    for seed in range(4):
        new_x, new_u = _logits(rows, vocab, torch.bfloat16, 41 + seed)
        x.copy_(new_x)
        u.copy_(new_u)
        graph.replay()
        want = sample_tokens(x, u, **settings)
        torch.cuda.synchronize()
        assert torch.equal(tokens, want[0]) and torch.equal(logs, want[1])
    other = [t.to(cuda) for t in _logits(rows, vocab, torch.bfloat16, 50)]
    want = [sample_tokens(x, u, **settings), sample_tokens(*other, **settings)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for stream, given in zip(streams, ((x, u), other)):
            with torch.cuda.stream(stream):
                got.append(sample_tokens(*given, **settings))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_shares_are_those_of_the_distribution(cuda):
    """200000 draws from 8 tokens: each one's share is within 5 standard deviations."""
    n, p = 200000, torch.tensor([0.4, 0.2, 0.15, 0.1, 0.08, 0.04, 0.02, 0.01], dtype=torch.float64)
    x = p.log().float().expand(n, 8).contiguous().to(cuda)
    u = torch.rand(n, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda, dtype=torch.float64)
    tokens, _ = sample_tokens(x, u)
    share = torch.bincount(tokens, minlength=8).double().cpu() / n
    assert bool(((share - p).abs() < 5 * (p * (1 - p) / n).sqrt()).all())


def test_tensors_that_do_not_fit_are_refused(cuda):
    x, u = torch.zeros(3, 10, device=cuda), torch.zeros(3, device=cuda)
    f = torch.zeros(3, device=cuda)
    for bad in (dict(logits=x[0]), dict(logits=x.t()), dict(logits=x.double()), dict(uniforms=u[:2]), dict(uniforms=u.half()), dict(uniforms=u.cpu()),
                dict(temperature=f.double()), dict(top_k=f), dict(top_k=f.long()), dict(top_p=f[:2]), dict(min_p=f.cpu()),
                dict(temperature=math.nan), dict(top_k=2 ** 31), dict(logits=x[:, :0]), dict(logits=x[:1].expand(3, 10))):
        with pytest.raises(ValueError):
            sample_tokens(**dict(dict(logits=x, uniforms=u), **bad))


@pytest.mark.parametrize("top_k", [1.5, 0.5, -0.1, math.inf, -math.inf, 2.0 ** 31, 10 ** 30])
def test_numbers_that_are_no_count_are_refused(cuda, top_k):
    x, u = torch.zeros(3, 10, device=cuda), torch.zeros(3, device=cuda)
    with pytest.raises(ValueError, match="whole number"):
        sample_tokens(x, u, top_k=top_k)
    assert sample_tokens(x, u, top_k=4.0)[0].tolist() == sample_tokens(x, u, top_k=4)[0].tolist()
