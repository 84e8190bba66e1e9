"""The sampler against its definition in whole numbers on the host: tokens are equal, not close.

The weights round(2^31 exp((x - max) / T)) are formed from f32 exponentials of the same function on
the same device; everything after them is integers, and two products in f64 that both sides round
alike.
"""

from __future__ import annotations

import math

import pytest
import torch

import tropnn_b200

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _row(value, n):
    return value.tolist() if isinstance(value, torch.Tensor) else [value] * n


def _f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


def _reference(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows, vocab = logits.shape
    x_dev = logits.detach().float()
    settings = zip(_row(temperature, rows), _row(top_k, rows), _row(top_p, rows), _row(min_p, rows), uniforms.tolist())
    tokens = []
    for n, (T, k, p, floor, u) in enumerate(settings):
        x = x_dev[n].cpu()
        if bool(x.isnan().any()) or float(x.max()) == -math.inf:
            tokens.append(-1)
            continue
        order = torch.sort(x, descending=True, stable=True).indices
        if not T > 0:
            tokens.append(int(order[0]))
            continue
        best = x_dev[n].max()
        inverse = 1.0 / torch.tensor(T, dtype=torch.float32, device=logits.device)
        e = torch.where(x_dev[n] == best, torch.ones_like(best), torch.exp((x_dev[n] - best) * inverse))
        e = torch.where(x_dev[n] == -math.inf, torch.zeros_like(e), e).cpu()
        weight = torch.round(e.double() * 2.0**31).long()[order]
        keep = torch.ones(vocab, dtype=torch.bool)
        if k > 0:
            keep[k:] = False
        kept = weight * keep
        before = torch.cumsum(kept, 0) - kept
        keep &= before.double() < _f32(p) * float(int(kept.sum()))
        keep &= e[order] >= _f32(floor)
        keep[0] = True
        back = torch.zeros(vocab, dtype=torch.int64).scatter_(0, order, weight * keep)
        upto = torch.cumsum(back, 0)
        total = int(upto[-1])
        target = min(int(math.floor(u * float(total))), total - 1)
        tokens.append(int((upto <= target).sum()))
    return torch.tensor(tokens)


def _inputs(rows, vocab, dtype, seed, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    logits = spread * torch.randn(rows, vocab, generator=gen)
    logits[:, :: max(1, vocab // 5)] += 5.0
    return logits.to(dtype).cuda(), torch.rand(rows, generator=gen).cuda()


SETTINGS = [
    {},
    {"temperature": 0.7},
    {"temperature": 0.0},
    {"top_k": 1},
    {"top_k": 40, "temperature": 1.3},
    {"top_p": 0.9},
    {"top_p": 0.5, "temperature": 2.0},
    {"min_p": 0.05},
    {"top_k": 500, "top_p": 0.95, "min_p": 0.01, "temperature": 0.9},
    {"top_k": 3, "top_p": 0.99},
    {"top_p": 0.0},
    {"min_p": 1.0},
    {"top_p": 0.9999, "temperature": 5.0},
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "vocab"), [(1, 1), (3, 2), (9, 47), (5, 1000), (4, 4097), (3, 32000), (2, 50001), (2, 131072)])
@pytest.mark.parametrize("settings", SETTINGS)
def test_tokens(rows, vocab, dtype, settings) -> None:
    logits, u = _inputs(rows, vocab, dtype, 3 * vocab + rows)
    got = tropnn_b200.sample_tokens_b200(logits, u, **settings)
    assert got.dtype == torch.int64
    assert torch.equal(got.cpu(), _reference(logits, u, **settings))


def test_a_large_vocabulary() -> None:
    logits, u = _inputs(2, 600_011, torch.float32, 4)
    for settings in ({}, {"top_p": 0.8}, {"top_k": 2000}):
        assert torch.equal(tropnn_b200.sample_tokens_b200(logits, u, **settings).cpu(), _reference(logits, u, **settings))


def _compare_some(logits, u, settings, some) -> None:
    """Some rows of a batch against the definition, and against each of them alone."""
    got = tropnn_b200.sample_tokens_b200(logits, u, **settings)
    pick = lambda v: v[some] if isinstance(v, torch.Tensor) else v  # noqa: E731
    want = _reference(logits[some], u[some], **{name: pick(v) for name, v in settings.items()})
    assert torch.equal(got[some].cpu(), want), settings
    for n in some[:2]:
        one = {name: v[n : n + 1] if isinstance(v, torch.Tensor) else v for name, v in settings.items()}
        alone = tropnn_b200.sample_tokens_b200(logits[n : n + 1], u[n : n + 1], **one)
        assert int(alone) == int(got[n]), settings


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [9001, 70001])
def test_more_rows_than_the_gpu_holds(vocab, dtype) -> None:
    """Rows that are streamed, a CTA each (of more than 2^16 tokens, or fewer), at odd offsets."""
    rows = 330
    whole, u = _inputs(rows, vocab + 2, dtype, vocab, spread=1.5)
    logits = whole[:, 1 : vocab + 1]
    logits[7] = logits[7].round()  # many tokens of one logit
    logits[8, 100:] = -math.inf
    logits[9] = -math.inf
    logits[10, vocab - 1] = float("nan")
    some = [3, 328, 7, 8, 9, 10, 200]
    for settings in ({"top_p": 0.9}, {"top_p": 0.9999, "temperature": 3.0}, {"top_k": 50}, {"top_k": 3000, "top_p": 0.9, "min_p": 0.001},
                     {"top_k": 1}, {}, {"min_p": 0.05}, {"temperature": 0.0}):
        _compare_some(logits, u, settings, some)
    gen = torch.Generator().manual_seed(12)
    pick = lambda values, t: torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=gen)].to(t).cuda()  # noqa: E731
    for _ in range(3):
        settings = {
            "temperature": pick([0.0, 0.6, 1.0, 1.5], torch.float32),
            "top_k": pick([0, 1, 20, 1000], torch.int32),
            "top_p": pick([1.0, 0.8, 0.99], torch.float32),
            "min_p": pick([0.0, 0.01, 0.2], torch.float32),
        }
        _compare_some(logits, u, settings, some)


@pytest.mark.parametrize(("dtype", "vocab"), [(torch.float32, 2_300_001), (torch.bfloat16, 4_600_003), (torch.float16, 4_600_003)])
def test_rows_of_more_batches_than_maxima_are_kept_for(dtype, vocab) -> None:
    logits, u = _inputs(1, vocab, dtype, 20)
    for settings in ({}, {"top_k": 50}, {"top_p": 0.9}, {"top_k": 5000, "top_p": 0.7}, {"min_p": 0.1}, {"temperature": 0.0}):
        assert torch.equal(tropnn_b200.sample_tokens_b200(logits, u, **settings).cpu(), _reference(logits, u, **settings))


@pytest.mark.parametrize("dtype", DTYPES)
def test_settings_of_each_row(dtype) -> None:
    rows, vocab = 64, 5003
    logits, u = _inputs(rows, vocab, dtype, 5)
    gen = torch.Generator().manual_seed(6)
    pick = lambda values, t: torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=gen)].to(t).cuda()  # noqa: E731
    settings = {
        "temperature": pick([0.0, -1.0, 0.5, 1.0, 1.5], torch.float32),
        "top_p": pick([1.0, 0.9, 0.3, 0.0], torch.float32),
        "min_p": pick([0.0, 0.02, 0.5], torch.float32),
    }
    for k_type in (torch.int32, torch.int64):
        settings["top_k"] = pick([0, -3, 1, 7, 300, 10**6], k_type)
        got = tropnn_b200.sample_tokens_b200(logits, u, **settings)
        assert torch.equal(got.cpu(), _reference(logits, u, **settings))


@pytest.mark.parametrize("settings", [{}, {"top_p": 0.6}, {"top_k": 25}, {"top_k": 30, "top_p": 0.5}, {"min_p": 0.3}])
def test_tokens_come_as_often_as_they_should(settings) -> None:
    """Evenly spaced uniforms over one distribution: a token's count is its probability times the
    number of rows, but for one row at either end of its stretch."""
    n, vocab = 4096, 61
    row = 1.5 * torch.randn(vocab, generator=torch.Generator().manual_seed(7)).cuda()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens = tropnn_b200.sample_tokens_b200(row.expand(n, vocab), u, **settings)
    counts = torch.bincount(tokens, minlength=vocab).cpu().double()
    p = torch.softmax(row.double().cpu(), 0)
    order = torch.sort(p, descending=True).indices
    keep = torch.ones(vocab, dtype=torch.bool)
    if "top_k" in settings:
        keep[settings["top_k"] :] = False
    ranked = p[order] * keep
    if "top_p" in settings:
        keep &= torch.cumsum(ranked, 0) - ranked < settings["top_p"] * ranked.sum()
    if "min_p" in settings:
        keep &= p[order] >= settings["min_p"] * p.max()
    want = torch.zeros(vocab, dtype=torch.float64).scatter_(0, order, p[order] * keep)
    want = want / want.sum() * n
    assert bool(((counts - want).abs() <= 1.0).all())
    assert not bool(counts[want == 0].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_index(dtype) -> None:
    vocab = 9001
    logits = torch.zeros(6, vocab, device="cuda", dtype=dtype)
    u = torch.tensor([0.0, 0.25, 0.5, 0.9, 0.9999, 1.0 - 2.0**-24], device="cuda")
    for settings in ({}, {"top_k": 100}, {"top_p": 0.1}, {"top_k": 5000, "top_p": 0.5}, {"temperature": 0.0}, {"min_p": 1.0}):
        assert torch.equal(tropnn_b200.sample_tokens_b200(logits, u, **settings).cpu(), _reference(logits, u, **settings))
    logits[:, 17] = -0.0  # as high as the zeros
    few = tropnn_b200.sample_tokens_b200(logits, u, top_k=18)
    assert torch.equal(few.cpu(), _reference(logits, u, top_k=18))
    # many tokens in a handful of levels: cuts inside a level
    coarse = (torch.randn(6, vocab, generator=torch.Generator().manual_seed(8)) * 2).round().to(dtype).cuda()
    for settings in ({"top_k": 50}, {"top_k": 4000}, {"top_p": 0.7}, {"top_p": 0.97, "top_k": 3000}):
        assert torch.equal(tropnn_b200.sample_tokens_b200(coarse, u, **settings).cpu(), _reference(coarse, u, **settings))


def test_neighbouring_values_in_f32() -> None:
    """Logits that differ in their last bits only: the ranking still goes by the logit."""
    gen = torch.Generator().manual_seed(9)
    steps = torch.randperm(3000, generator=gen).int()
    logits = (torch.full((3000,), 5.0).view(torch.int32) - steps).view(torch.float32).expand(4, 3000).contiguous().cuda()
    u = torch.rand(4, generator=gen).cuda()
    tiny = (1e-30 * torch.randn(4, 3000, generator=gen)).cuda()
    for x in (logits, tiny):
        for settings in ({"top_k": 20}, {"top_k": 1500}, {"top_p": 0.33}, {"temperature": 0.0}):
            assert torch.equal(tropnn_b200.sample_tokens_b200(x, u, **settings).cpu(), _reference(x, u, **settings))


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows(dtype) -> None:
    """-inf is never drawn; a row of nothing else, or with a NaN, gives -1; +inf takes everything; the
    type's lowest value is a value."""
    logits, u = _inputs(7, 800, dtype, 10)
    logits[0, 5:] = -math.inf
    logits[1] = -math.inf
    logits[2, 400] = float("nan")
    logits[3, 300] = logits[3, 700] = math.inf
    logits[4] = torch.finfo(dtype).min
    logits[5] = -math.inf
    logits[5, 123] = torch.finfo(dtype).min
    u[:] = 0.75
    for settings in ({}, {"top_k": 600}, {"top_p": 0.999}, {"temperature": 0.0}, {"temperature": 1e-30}, {"temperature": 1e30}):
        got = tropnn_b200.sample_tokens_b200(logits, u, **settings).cpu()
        assert torch.equal(got, _reference(logits, u, **settings)), settings
        assert int(got[0]) < 5 and int(got[1]) == int(got[2]) == -1
        assert int(got[3]) in (300, 700) and int(got[5]) == 123


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_temperatures_whose_inverse_is_subnormal(dtype) -> None:
    lowest = torch.finfo(dtype).min
    logits = torch.tensor([0.0, lowest, lowest / 2, lowest / 4, -1.0, -math.inf, lowest / 3], dtype=dtype).cuda().expand(64, 7)
    u = ((torch.arange(64) + 0.5) / 64).cuda()
    for settings in ({"temperature": 1e38}, {"temperature": 3.3e38}, {"temperature": 3e38, "top_p": 0.8}, {"temperature": 2e38, "top_k": 4}):
        got = tropnn_b200.sample_tokens_b200(logits, u, **settings)
        assert torch.equal(got.cpu(), _reference(logits, u, **settings)), settings


def test_uniforms_at_the_ends() -> None:
    logits = torch.randn(5, 300, generator=torch.Generator().manual_seed(11)).cuda()
    u = torch.tensor([0.0, 1.0, 1.0 - 2.0**-24, -0.5, 2.0], device="cuda")
    got = tropnn_b200.sample_tokens_b200(logits, u).tolist()
    assert got == [0, 299, 299, 0, 299]


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_do_not_change_a_token(dtype) -> None:
    whole = (2.0 * torch.randn(3, 4, 2051, generator=torch.Generator().manual_seed(12))).to(dtype).cuda()
    u = torch.rand(3, 4, generator=torch.Generator().manual_seed(13)).cuda()
    for vocab in (2000, 2001, 2051):
        settings = {"top_p": 0.9, "top_k": 700}
        last = tropnn_b200.sample_tokens_b200(whole[:, -1, :vocab], u[:, -1], **settings)
        assert torch.equal(last.cpu(), _reference(whole[:, -1, :vocab], u[:, -1], **settings))
        both = tropnn_b200.sample_tokens_b200(whole[:, ::2, :vocab], u[:, ::2], **settings)
        flat = whole[:, ::2, :vocab].reshape(6, vocab)
        assert torch.equal(both.cpu().view(-1), _reference(flat, u[:, ::2].reshape(6), **settings))
        # each row alone, and shifted within memory
        for n in range(3):
            alone = tropnn_b200.sample_tokens_b200(whole[n, -1, :vocab].clone(), u[n, -1], **settings)
            assert alone.shape == () and int(alone) == int(last[n])
    turned = whole[0].t()[:, :2].t()  # no copy needed
    tokens = tropnn_b200.sample_tokens_b200(turned, u[0, :2])
    assert torch.equal(tokens.cpu(), _reference(turned, u[0, :2]))
    scattered = whole[0, :2].t().contiguous().t()  # the vocabulary is not the fast dimension
    assert torch.equal(tropnn_b200.sample_tokens_b200(scattered, u[0, :2]), tokens)


def test_offsets_past_32_bits() -> None:
    far = (1 << 31) + 8
    store = torch.zeros(far + 4096, dtype=torch.float16, device="cuda")
    view = store.as_strided((2, 1003), (far, 1))
    logits, u = _inputs(2, 1003, torch.float16, 14)
    view.copy_(logits)
    assert torch.equal(tropnn_b200.sample_tokens_b200(view, u, top_p=0.9).cpu(), _reference(logits, u, top_p=0.9))


def test_side_stream_and_no_rows() -> None:
    logits, u = _inputs(4, 3001, torch.bfloat16, 15)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = tropnn_b200.sample_tokens_b200(logits, u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got.cpu(), _reference(logits, u, top_p=0.9))
    assert tropnn_b200.sample_tokens_b200(torch.empty(0, 9, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)


def test_refusals() -> None:
    op = tropnn_b200.sample_tokens_b200
    x, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    for call in (
        lambda: op(x, u[:1]),
        lambda: op(x, u.cpu()),
        lambda: op(x[:, :0], u),
        lambda: op(x, u, temperature=-0.5),
        lambda: op(x, u, temperature=float("nan")),
        lambda: op(x, u, top_k=-1),
        lambda: op(x, u, top_p=1.5),
        lambda: op(x, u, min_p=-0.1),
        lambda: op(x, u, top_p=torch.ones(3, device="cuda")),
        lambda: op(x, u, top_k=torch.ones(1, dtype=torch.int32, device="cuda")),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (
        lambda: op(x.double(), u),
        lambda: op(x, u.double()),
        lambda: op(x, u, temperature=torch.ones(2, dtype=torch.float64, device="cuda")),
        lambda: op(x, u, top_k=torch.ones(2, device="cuda")),
    ):
        with pytest.raises(TypeError):
            call()
