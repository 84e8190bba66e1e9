"""The distillation loss and its gradient against the formulas in f64.

Tolerances: exponentials are good to about 2^-22 and differences from the row's maximum (below 40
here) to 40 * 2^-24, so a probability is within 4e-6 of itself and a logarithm within 4e-6: 1e-5
of (1 + T^2) (1 + loss) for a loss. A gradient entry is a sum of probabilities: within 1e-5 of their
sum times its weights, and the rounding of its type (2^-24, 2^-11 and half of f16's smallest step
2^-25, 2^-8) of its value.
"""

from __future__ import annotations

import math

import pytest
import torch

import tropnn_b200

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _reference(logits, teacher, indices, labels, T, w, ignore=-100):
    """(losses, gradient of each loss, sum of the probabilities in each gradient entry, valid), f64."""
    x = logits.detach().double().cpu()
    t, at = teacher.double().cpu(), indices.long().cpu()
    rows, vocab = x.shape
    losses, valid = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.bool)
    grad, mass = torch.zeros_like(x), torch.zeros_like(x)
    for n in range(rows):
        there = (at[n] >= 0) & (at[n] < vocab) & (t[n] != -math.inf)
        if w < 1 and bool(there.any()):
            i = at[n][there]
            q = torch.softmax(t[n][there] / T, dim=0)
            log_q = torch.log_softmax(t[n][there] / T, dim=0)
            log_p = torch.log_softmax(x[n] / T, dim=0)
            terms = torch.where(q > 0, q * (log_q - log_p[i]), torch.zeros_like(q))
            losses[n] += (1 - w) * T * T * terms.sum()
            spread = torch.zeros(vocab, dtype=torch.float64).index_add_(0, i, q)
            grad[n] += (1 - w) * T * (log_p.exp() - spread)
            mass[n] += (1 - w) * T * (log_p.exp() + spread)
            valid[n] = True
        y = -1 if labels is None else int(labels[n])
        if w > 0 and y != ignore and 0 <= y < vocab:
            log_p = torch.log_softmax(x[n], dim=0)
            losses[n] -= w * log_p[y]
            one = torch.zeros(vocab, dtype=torch.float64)
            one[y] = 1.0
            grad[n] += w * (log_p.exp() - one)
            mass[n] += w * (log_p.exp() + one)
            valid[n] = True
    return losses, grad, mass, valid


def _close_loss(got, want, T):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    assert bool(((got - want).abs() <= 1e-5 * (1 + T * T) * (1 + want.abs())).all()), float((got - want).abs().max())


def _close_grad(got, grad, mass, scale, dtype):
    got = got.detach().double().cpu()
    want = grad * scale
    bound = UNIT[dtype] * want.abs() + 1e-5 * mass * scale.abs() + (2.0**-25 if dtype == torch.float16 else 1e-30)
    assert got.shape == want.shape
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())


def _inputs(rows, vocab, top, dtype, seed, ragged=True, teacher_dtype=None):
    gen = torch.Generator().manual_seed(seed)
    logits = 2.0 * torch.randn(rows, vocab, generator=gen)
    at = torch.stack([torch.randperm(vocab, generator=gen)[:top] for _ in range(rows)]) if rows else torch.zeros(0, top).long()
    teacher = 2.5 * torch.randn(rows, top, generator=gen) + 4.0
    logits.scatter_add_(1, at, 0.7 * teacher)
    labels = torch.randint(0, vocab, (rows,), generator=gen)
    if rows and top:
        labels[::2] = at[::2, 0]
    if ragged and rows:
        count = torch.randint(0, top + 1, (rows,), generator=gen)
        at = torch.where(torch.arange(top) < count[:, None], at, torch.full_like(at, -1))
        labels[torch.rand(rows, generator=gen) < 0.3] = -100
    return logits.to(dtype).cuda(), teacher.to(teacher_dtype or dtype).cuda(), at.cuda(), labels.cuda()


SHAPES = [  # rows, vocab, top
    (1, 1, 1),
    (3, 2, 2),
    (17, 47, 8),
    (5, 1000, 20),
    (4, 4097, 64),
    (3, 32000, 1),
    (2, 50001, 128),
    (2, 131072, 64),
    (1, 262147, 5),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize(("T", "w"), [(1.0, 0.0), (2.0, 0.3), (1.0, 0.5), (3.0, 0.0), (2.0, 1.0)])
def test_loss_and_gradient(shape, dtype, T, w) -> None:
    rows, vocab, top = shape
    logits, teacher, at, labels = _inputs(rows, vocab, top, dtype, vocab + top)
    losses, grad, mass, valid = _reference(logits, teacher, at, labels, T, w)
    args = dict(temperature=T, label_weight=w)
    # in one call, a scale a row
    scale = 0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(3))
    got, got_grad = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, row_scale=scale.cuda(), **args)
    _close_loss(got, losses, T)
    assert got_grad.dtype == dtype and got_grad.is_contiguous()
    _close_grad(got_grad, grad, mass, scale.double()[:, None], dtype)
    # through autograd, each reduction
    leaf = logits.detach().requires_grad_()
    count = max(1, int(valid.sum()))
    for reduction, total, each in (("mean", losses.sum() / count, 1.0 / count), ("sum", losses.sum(), 1.0)):
        loss = tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, reduction=reduction, **args)
        _close_loss(loss, total, T * (1 if reduction == "mean" else math.sqrt(rows)))
        (g,) = torch.autograd.grad(loss, leaf, torch.tensor(3.0, device="cuda"))
        _close_grad(g, grad, mass, torch.full((rows, 1), 3.0 * each, dtype=torch.float64), dtype)
    loss = tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, reduction="none", **args)
    _close_loss(loss, losses, T)
    (g,) = torch.autograd.grad(loss, leaf, scale.cuda())
    _close_grad(g, grad, mass, scale.double()[:, None], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize(("T", "w"), [(1.5, 0.3), (0.7, 0.5), (4.0, 0.25)])
def test_labels_at_a_temperature_of_its_own(shape, dtype, T, w) -> None:
    """Two sums an element whose exponentials have nothing to do with one another."""
    test_loss_and_gradient(shape, dtype, T, w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_exponentials_of_the_labels(dtype) -> None:
    """A row with a label alone has the gradient w p1, here relative to its largest entry w / sum: a
    power of two to 2^-22 of it, its argument d log2(e) to 1.5 * 2^-24 of that (the product and the
    constant), and two roundings of 2^-24, in the type that it is stored in."""
    vocab = 4096
    logits = torch.linspace(-75.0, 0.0, vocab, dtype=torch.float64).to(dtype)
    logits = torch.stack([logits, logits.flip(0), logits.roll(1), logits.roll(3)]).cuda()  # each place in a vector
    label = 5
    at = torch.full((4, 1), -1, dtype=torch.int64, device="cuda")
    _, grad = tropnn_b200.distill_loss_grad_b200(
        logits, torch.zeros(4, 1, device="cuda"), at, torch.full((4,), label, device="cuda"), temperature=1.5, label_weight=0.5)
    x, g = logits.double().cpu(), grad.double().cpu()
    want = x.exp()
    rest = torch.arange(vocab) != label
    ratio = g / g.amax(dim=1, keepdim=True)
    bound = 2.0**-22 + 1.5 * 2.0**-24 * x.abs() + 3 * 2.0**-24 + 2 * (UNIT[dtype] if dtype != torch.float32 else 0.0)
    assert bool(((ratio / want - 1).abs() <= bound)[:, rest].all()), float(((ratio / want - 1).abs() - bound)[:, rest].max())


@pytest.mark.parametrize("top", [129, 500, 1024])
@pytest.mark.parametrize(("T", "w"), [(1.0, 0.0), (2.0, 0.3), (1.5, 0.4)])
def test_long_teacher_lists(top, T, w) -> None:
    """More than 128 entries are read by several warps: entries of one index in the shares of two, the
    label among them, shares without an entry."""
    logits, teacher, at, labels = _inputs(6, 5003, top, torch.float32, 31 + top, ragged=False)
    at[:, top - 1] = at[:, 0]
    at[:, 128] = at[:, 127]
    labels[:3] = at[:3, 0]
    labels[3] = at[3, top - 1]
    labels[4] = -100
    at[4, :128] = -1  # the first share has none
    at[5, 1:] = -1
    teacher[2, 64:] -= 200.0  # shares that weigh nothing
    losses, grad, mass, _ = _reference(logits, teacher, at, labels, T, w)
    got, got_grad = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, temperature=T, label_weight=w)
    _close_loss(got, losses, T)
    _close_grad(got_grad, grad, mass, torch.ones(6, 1, dtype=torch.float64), torch.float32)
    leaf = logits.detach().requires_grad_()
    loss = tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, temperature=T, label_weight=w, reduction="none")
    _close_loss(loss, losses, T)
    (got_grad,) = torch.autograd.grad(loss.sum(), leaf)
    _close_grad(got_grad, grad, mass, torch.ones(6, 1, dtype=torch.float64), torch.float32)


@pytest.mark.parametrize(("dtype", "vocab"), [(torch.float32, 450_001), (torch.bfloat16, 900_001), (torch.float16, 850_006)])
@pytest.mark.parametrize(("T", "w"), [(1.0, 0.0), (2.0, 0.3), (1.5, 0.4)])
def test_rows_that_shared_memory_does_not_hold(dtype, vocab, T, w) -> None:
    logits, teacher, at, labels = _inputs(2, vocab, 40, dtype, 32, ragged=False)
    losses, grad, mass, _ = _reference(logits, teacher, at, labels, T, w)
    got, got_grad = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, temperature=T, label_weight=w)
    _close_loss(got, losses, T)
    _close_grad(got_grad, grad, mass, torch.ones(2, 1, dtype=torch.float64), dtype)


@pytest.mark.parametrize(("rows", "vocab", "dtype"), [(900, 3001, torch.float16), (115, 131072, torch.bfloat16), (460, 16001, torch.float32)])
def test_more_rows_than_the_gpu_holds(rows, vocab, dtype) -> None:
    """And a few of the rows by themselves: the sums' order may differ with the rows' number, so as close
    to the formulas, not bit for bit."""
    logits, teacher, at, labels = _inputs(rows, vocab, 16, dtype, 33)
    args = dict(temperature=1.5, label_weight=0.25)
    losses, grad, mass, _ = _reference(logits, teacher, at, labels, 1.5, 0.25)
    got, got_grad = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, **args)
    _close_loss(got, losses, 1.5)
    _close_grad(got_grad, grad, mass, torch.ones(rows, 1, dtype=torch.float64), dtype)
    some = slice(rows - 4, rows - 1)
    got, got_grad = tropnn_b200.distill_loss_grad_b200(logits[some], teacher[some], at[some], labels[some], **args)
    _close_loss(got, losses[some], 1.5)
    _close_grad(got_grad, grad[some], mass[some], torch.ones(3, 1, dtype=torch.float64), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize(("T", "w"), [(0.5, 0.0), (0.5, 0.3), (0.25, 0.5), (2.0, 0.3)])
def test_teacher_entries_of_the_lowest_value(dtype, T, w) -> None:
    """A logit of the type's lowest value is a value, below T = 1 too: alone it is a uniform teacher,
    beside others it weighs nothing."""
    for top in (6, 300):
        logits, teacher, at, labels = _inputs(3, 777, top, torch.float32, 34, ragged=False, teacher_dtype=dtype)
        teacher[0] = torch.finfo(dtype).min
        teacher[1, 2:] = torch.finfo(dtype).min
        losses, grad, mass, _ = _reference(logits, teacher, at, labels, T, w)
        got, got_grad = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, temperature=T, label_weight=w)
        _close_loss(got, losses, T)
        _close_grad(got_grad, grad, mass, torch.ones(3, 1, dtype=torch.float64), torch.float32)
        leaf = logits.detach().requires_grad_()
        loss = tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, temperature=T, label_weight=w, reduction="none")
        _close_loss(loss, losses, T)
        _close_grad(torch.autograd.grad(loss.sum(), leaf)[0], grad, mass, torch.ones(3, 1, dtype=torch.float64), torch.float32)


def test_gradient_against_differences() -> None:
    """Along a random direction; f32 losses of about 3 are good to 1e-6, over a step of 1e-2: 1e-4."""
    logits, teacher, at, labels = _inputs(6, 500, 16, torch.float32, 21)
    args = dict(temperature=2.0, label_weight=0.4)
    way = torch.randn(6, 500, generator=torch.Generator().manual_seed(1)).cuda()
    leaf = logits.clone().requires_grad_()
    (grad,) = torch.autograd.grad(tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, **args), leaf)
    eps = 1e-2
    ends = [tropnn_b200.distill_loss_b200(logits + e * way, teacher, at, labels, **args).double() for e in (eps, -eps)]
    slope = (grad.double() * way).sum()
    assert abs(float((ends[0] - ends[1]) / (2 * eps) - slope)) <= 1e-3 * (1 + abs(float(slope)))


def test_rows_without_a_target() -> None:
    """No entries and no label: loss 0, gradient 0, not counted, whatever the logits hold."""
    logits, teacher, at, labels = _inputs(5, 300, 4, torch.float32, 22, ragged=False)
    at[1] = -1
    labels[1] = -100
    at[2] = torch.tensor([300, 1 << 40, -5, 301])  # out of range: padding
    labels[2] = 300
    teacher[3] = -math.inf
    labels[3] = -7
    logits[1] = float("nan")
    logits[2] = -math.inf
    leaf = logits.clone().requires_grad_()
    for w in (0.0, 0.5):
        loss = tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, label_weight=w)
        (grad,) = torch.autograd.grad(loss, leaf)
        losses, want, mass, valid = _reference(logits, teacher, at, labels, 1.0, w)
        assert valid.tolist() == [True, False, False, False, True]
        _close_loss(loss, losses.sum() / 2, 1.0)
        assert not bool(grad[1:4].any())
        _close_grad(grad, want, mass, torch.full((5, 1), 0.5, dtype=torch.float64), torch.float32)
    nothing = torch.full_like(at, -1)
    loss = tropnn_b200.distill_loss_b200(leaf, teacher, nothing)
    (grad,) = torch.autograd.grad(loss, leaf)
    assert float(loss) == 0.0 and not bool(grad.any())
    none = tropnn_b200.distill_loss_b200(leaf, teacher[:, :0], nothing[:, :0], reduction="none")
    assert not bool(none.any())


def test_masked_logits() -> None:
    """-inf logits have probability 0 and gradient 0; under a teacher's entry the loss is infinite
    and the gradient still p - q; a whole row of them has no distribution."""
    logits, teacher, at, labels = _inputs(4, 64, 3, torch.float32, 23, ragged=False)
    logits[0, :] = torch.where(torch.isin(torch.arange(64, device="cuda"), torch.cat([at[0], labels[:1]])), logits[0], -math.inf)
    logits[1, at[1, 0]] = -math.inf
    logits[2] = -math.inf
    logits[3] = torch.finfo(torch.float32).min
    losses, grad = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, label_weight=0.25, temperature=2.0)
    want, want_grad, mass, _ = _reference(logits, teacher, at, labels, 2.0, 0.25)
    _close_loss(losses[0], want[0], 2.0)
    _close_grad(grad[:1], want_grad[:1], mass[:1], torch.ones(1, 1, dtype=torch.float64), torch.float32)
    off = (logits[0] == -math.inf).nonzero()[:, 0]
    assert not bool(grad[0, off].any())
    assert float(losses[1]) == math.inf
    spot = int(at[1, 0])
    q = torch.softmax(teacher[1].double() / 2.0, dim=0)[0]
    base = -0.75 * 2.0 * float(q) - (0.25 if int(labels[1]) == spot else 0.0)
    assert float(grad[1, spot]) == pytest.approx(base, rel=1e-5)
    assert math.isnan(float(losses[2])) and bool(grad[2].isnan().any())
    _close_loss(losses[3], want[3], 2.0)  # a row of the type's lowest value is a uniform one


def test_repeated_entries_add_up() -> None:
    logits, teacher, at, labels = _inputs(3, 40, 6, torch.float32, 24, ragged=False)
    at[:, 3] = at[:, 0]
    at[:, 4] = at[:, 0]
    labels[1] = at[1, 0]
    losses, grad = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, label_weight=0.5)
    want, want_grad, mass, _ = _reference(logits, teacher, at, labels, 1.0, 0.5)
    _close_loss(losses, want, 1.0)
    _close_grad(grad, want_grad, mass, torch.ones(3, 1, dtype=torch.float64), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_logits(dtype) -> None:
    """All tokens but the last of each sequence, out of a padded vocabulary, read in place."""
    gen = torch.Generator().manual_seed(25)
    whole = (2.0 * torch.randn(3, 6, 1009, generator=gen)).to(dtype).cuda()
    for vocab in (1000, 1001, 1009):
        view = whole[:, :-1, :vocab]
        at = torch.randint(0, vocab, (3, 5, 7), generator=gen).int().cuda()
        teacher = torch.randn(3, 5, 7, generator=gen).cuda()
        labels = torch.randint(0, vocab, (3, 5), generator=gen).int().cuda()
        leaf = view.detach().requires_grad_()
        assert leaf.stride() == view.stride()
        loss = tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, temperature=2.0, label_weight=0.5, reduction="sum")
        (grad,) = torch.autograd.grad(loss, leaf)
        flat = lambda t: t.reshape(15, *t.shape[2:])  # noqa: E731
        losses, want, mass, _ = _reference(flat(view), flat(teacher), flat(at), flat(labels), 2.0, 0.5)
        _close_loss(loss, losses.sum(), 8.0)
        _close_grad(flat(grad), want, mass, torch.ones(15, 1, dtype=torch.float64), dtype)
    # four dimensions, a transposed vocabulary, one row alone
    odd = whole.transpose(1, 2)[:, :, :2]  # [3, 1009, 2]: unit stride is elsewhere
    at = torch.zeros(3, 1009, 1, dtype=torch.int64, device="cuda")
    losses, _ = tropnn_b200.distill_loss_grad_b200(odd, torch.zeros(3, 1009, 1, device="cuda"), at)
    want = -torch.log_softmax(odd.double(), dim=-1)[..., 0].cpu()
    _close_loss(losses, want, 1.0)
    losses, grad = tropnn_b200.distill_loss_grad_b200(whole[0, 0], torch.zeros(1, device="cuda"), at[0, 0])
    assert losses.shape == () and grad.shape == (1009,)
    losses, _ = tropnn_b200.distill_loss_grad_b200(
        whole.view(3, 1, 6, 1009), torch.zeros(3, 1, 6, 1, device="cuda"), at[:, :6].view(3, 1, 6, 1))
    assert losses.shape == (3, 1, 6)


def test_ignore_index_inside_the_vocabulary() -> None:
    logits, teacher, at, labels = _inputs(8, 100, 4, torch.float32, 26)
    labels[:4] = 0
    loss = tropnn_b200.distill_loss_b200(logits, teacher, at, labels, label_weight=0.7, ignore_index=0, reduction="none")
    _close_loss(loss, _reference(logits, teacher, at, labels, 1.0, 0.7, ignore=0)[0], 1.0)


def test_scales_before_rounding() -> None:
    """A gradient far below f16's range survives when the loss scale comes in with the call."""
    logits, teacher, at, labels = _inputs(4, 20000, 8, torch.float16, 27, ragged=False)
    leaf = logits.detach().requires_grad_()
    loss = tropnn_b200.distill_loss_b200(leaf, teacher, at)
    (grad,) = torch.autograd.grad(loss * 65536.0, leaf)
    _, want, mass, _ = _reference(logits, teacher, at, None, 1.0, 0.0)
    _close_grad(grad, want, mass, torch.full((4, 1), 65536.0 / 4, dtype=torch.float64), torch.float16)
    _, fused = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, row_scale=65536.0 / 4)
    assert torch.equal(fused, grad)


def test_runs_are_bitwise_equal_and_rows_stand_alone() -> None:
    logits, teacher, at, labels = _inputs(9, 33000, 32, torch.bfloat16, 28)
    args = dict(temperature=2.0, label_weight=0.25, row_scale=0.125)
    a = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, **args)
    b = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, **args)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_side_stream_two_backwards_and_in_place_changes() -> None:
    logits, teacher, at, labels = _inputs(3, 5000, 8, torch.float32, 29)
    leaf = logits.clone().requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        loss = tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, label_weight=0.5)
        loss *= 2.0  # an ordinary tensor
        first = torch.autograd.grad(loss, leaf, retain_graph=True)[0]
        again = torch.autograd.grad(loss, leaf, retain_graph=True)[0]
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(first, again)
    at[0, 0] = 3
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, leaf)


@pytest.mark.parametrize("view", [False, True])
def test_saved_tensors_are_released_and_may_be_moved(view) -> None:
    """A loss that outlives its backward holds no logits, and saved tensors may come back elsewhere."""
    logits, teacher, at, labels = _inputs(64, 5000, 8, torch.bfloat16, 16)
    if view:
        logits = torch.cat([logits, logits], dim=1)[:, :5000]
    kw = dict(temperature=2.0, label_weight=0.25)
    leaf = logits.detach().requires_grad_()
    (want,) = torch.autograd.grad(tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, **kw), leaf)
    with torch.autograd.graph.save_on_cpu():
        loss = tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, **kw)
    junk = [torch.full_like(t, 1) for t in (logits, teacher, at, labels)]
    (got,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(got, want)
    del junk, loss

    before = torch.cuda.memory_allocated()
    student = leaf * 1.0
    loss = tropnn_b200.distill_loss_b200(student, teacher, at, labels, **kw)
    del student
    loss.backward()
    leaf.grad = None
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before <= 4096  # the loss itself


def test_offsets_past_32_bits() -> None:
    far = (1 << 31) + 8
    store = torch.zeros(far + 4096, dtype=torch.float16, device="cuda")
    view = store.as_strided((2, 1003), (far, 1))
    logits, teacher, at, labels = _inputs(2, 1003, 8, torch.float16, 30, ragged=False)
    view.copy_(logits)
    got = tropnn_b200.distill_loss_grad_b200(view, teacher, at, labels, label_weight=0.5)
    want = tropnn_b200.distill_loss_grad_b200(logits, teacher, at, labels, label_weight=0.5)
    _close_loss(got[0], _reference(logits, teacher, at, labels, 1.0, 0.5)[0], 1.0)
    _close_loss(got[0], want[0].double().cpu(), 1.0)


def test_no_rows() -> None:
    logits, at = torch.empty(0, 10, device="cuda", requires_grad=True), torch.empty(0, 3, dtype=torch.int64, device="cuda")
    loss = tropnn_b200.distill_loss_b200(logits, torch.empty(0, 3, device="cuda"), at)
    assert float(loss) == 0.0
    assert torch.autograd.grad(loss, logits)[0].shape == (0, 10)


def test_temperatures_that_f32_cannot_square_are_refused() -> None:
    logits, teacher, at, labels = _inputs(2, 50, 3, torch.float32, 35)
    for T in (1e-40, 1e-25, 1e25, 3e38):
        for op in (tropnn_b200.distill_loss_b200, tropnn_b200.distill_loss_grad_b200):
            with pytest.raises(ValueError, match="temperature"):
                op(logits, teacher, at, labels, temperature=T, label_weight=0.5)
            op(logits, teacher, at, labels, temperature=T, label_weight=1.0)  # the labels have none


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(grad_mode) -> None:
    """A tangent is not lost, which would be a derivative of 0."""
    logits, teacher, at, _ = _inputs(2, 50, 3, torch.float32, 36)
    scale = torch.ones(2, device="cuda")
    make = torch.autograd.forward_ad.make_dual
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        tropnn_b200.distill_loss_b200(logits, teacher, at)
        moved, moved_teacher = make(logits, torch.ones_like(logits)), make(teacher, torch.ones_like(teacher))
        for call in (
            lambda: tropnn_b200.distill_loss_b200(moved, teacher, at),
            lambda: tropnn_b200.distill_loss_b200(logits, moved_teacher, at),
            lambda: tropnn_b200.distill_loss_grad_b200(moved, teacher, at),
            lambda: tropnn_b200.distill_loss_grad_b200(logits, moved_teacher, at),
            lambda: tropnn_b200.distill_loss_grad_b200(logits, teacher, at, row_scale=make(scale, scale)),
        ):
            with pytest.raises(NotImplementedError):
                call()


def test_saved_tensors_may_come_back_with_other_strides() -> None:
    from .test_recurrence_gpu import _elsewhere

    logits, teacher, at, labels = _inputs(5, 700, 9, torch.float32, 37)
    leaf = logits.requires_grad_()
    kw = dict(temperature=2.0, label_weight=0.25)
    (want,) = torch.autograd.grad(tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, **kw), leaf)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _elsewhere):
        (got,) = torch.autograd.grad(tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, **kw), leaf)
    assert torch.equal(got, want)


def test_calls_in_a_cuda_graph() -> None:
    """Loss, gradient, both in one call and a draw captured once and replayed on other inputs."""
    logits, teacher, at, labels = _inputs(6, 3001, 9, torch.bfloat16, 38)
    leaf, u = logits.clone().requires_grad_(), torch.rand(6, generator=torch.Generator().manual_seed(1)).cuda()
    kw = dict(temperature=2.0, label_weight=0.25)

    def calls():
        loss = tropnn_b200.distill_loss_b200(leaf, teacher, at, labels, **kw)
        (grad,) = torch.autograd.grad(loss, leaf)
        tokens = tropnn_b200.sample_tokens_b200(leaf, u, top_k=40, top_p=0.9)
        return [loss.detach(), grad, *tropnn_b200.distill_loss_grad_b200(leaf.detach(), teacher, at, labels, **kw), tokens]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        calls()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    with torch.no_grad():
        leaf.copy_(logits.roll(1, dims=0))
        teacher.neg_()
        u.copy_(1 - u)
    graph.replay()
    got = [t.clone() for t in out]
    assert all(torch.equal(a, b) for a, b in zip(got, calls()))


def test_refusals() -> None:
    op = tropnn_b200.distill_loss_b200
    x, t = torch.zeros(2, 9, device="cuda"), torch.zeros(2, 3, device="cuda")
    at, y = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for call in (
        lambda: op(x, t[:1], at),
        lambda: op(x, t, at[:, :2]),
        lambda: op(x, t, at, y[:1]),
        lambda: op(x, t.cpu(), at),
        lambda: op(x, t, at, temperature=0.0),
        lambda: op(x, t, at, temperature=float("inf")),
        lambda: op(x, t, at, label_weight=0.5),
        lambda: op(x, t, at, y, label_weight=1.5),
        lambda: op(x, t, at, reduction="batchmean"),
        lambda: op(x[:, :0], t, at),
        lambda: op(x, torch.zeros(2, 1025, device="cuda"), torch.zeros(2, 1025, dtype=torch.int64, device="cuda")),
        lambda: tropnn_b200.distill_loss_grad_b200(x, t, at, row_scale=torch.zeros(3, device="cuda")),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (
        lambda: op(x.double(), t, at),
        lambda: op(x, t.double(), at),
        lambda: op(x, t, at.float()),
        lambda: op(x, t, at, y.float()),
        lambda: tropnn_b200.distill_loss_grad_b200(x, t, at, row_scale=torch.zeros(2, device="cuda").half()),
    ):
        with pytest.raises(TypeError):
            call()
