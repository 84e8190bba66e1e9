"""The gated recurrence against the same steps in f64, one after the other.

Tolerances: the state is f32 and a step rounds it by a few parts in 2^24, which the gates then
forget as fast as the state itself, so h stays within 1e-5 of its sequence's largest value, and
the gradients, sums of the same kind, within 1e-5 of theirs. A 16-bit output adds its rounding:
2^-11 (f16, and half its smallest step 2^-25) or 2^-8 (bf16) of the value.
"""

from __future__ import annotations

import pytest
import torch

import tropnn_b200

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 0.0, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _reference(gate, value, h0, reset, grad=None, grad_last=None):
    f, x = gate.detach().double().cpu(), value.detach().double().cpu()
    batch, steps, dim = f.shape
    h = torch.zeros(batch, dim, dtype=torch.float64) if h0 is None else h0.detach().double().cpu().clone()
    cut = torch.zeros(batch, steps, dtype=torch.bool) if reset is None else reset.bool().cpu()
    a, c = torch.sigmoid(f), torch.sigmoid(-f)
    hs, before = torch.empty_like(x), torch.empty_like(x)
    for t in range(steps):
        before[:, t] = torch.where(cut[:, t, None], torch.zeros_like(h), h)
        h = a[:, t] * before[:, t] + c[:, t] * x[:, t]
        hs[:, t] = h
    if grad is None:
        return hs, h
    r = torch.zeros(batch, dim, dtype=torch.float64) if grad_last is None else grad_last.double().cpu().clone()
    df, dx = torch.empty_like(x), torch.empty_like(x)
    for t in reversed(range(steps)):
        ds = grad[:, t].double().cpu() + r
        dx[:, t] = c[:, t] * ds
        df[:, t] = ds * (before[:, t] - x[:, t]) * a[:, t] * c[:, t]
        r = torch.where(cut[:, t, None], torch.zeros_like(ds), a[:, t] * ds)
    return hs, h, df, dx, r


def _close(got, want, dtype):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    if want.numel() == 0:
        return
    bound = 1e-5 * want.abs().max() + UNIT[dtype] * want.abs() + (2.0**-25 if dtype == torch.float16 else 0.0)
    assert bool((got - want).abs().le(bound).all()), float(((got - want).abs() - bound).max())


def _inputs(batch, steps, dim, dtype, seed, fused=False):
    gen = torch.Generator().manual_seed(seed)
    bias = 2.0 + 1.5 * torch.randn(dim, generator=gen)
    gate = torch.randn(batch, steps, dim, generator=gen) + bias
    value = torch.randn(batch, steps, dim, generator=gen)
    if fused:
        both = torch.cat([gate, value], dim=2).to(dtype).cuda()
        return both[..., :dim], both[..., dim:], torch.randn(batch, dim, generator=gen).cuda()
    return gate.to(dtype).cuda(), value.to(dtype).cuda(), torch.randn(batch, dim, generator=gen).cuda()


SHAPES = [
    (1, 1, 1),
    (2, 1, 64),
    (3, 7, 5),
    (2, 63, 65),  # one less than a saved tile, one channel past a block
    (1, 64, 66),
    (2, 65, 128),
    (3, 129, 31),
    (1, 1000, 130),
    (5, 1025, 64),
    (1, 4099, 16),  # a long one, few channels
    (40, 130, 200),
    (2, 20011, 24),  # so few channels that the sequence is cut into chunks
    (1, 20011, 21),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("fused", [False, True])
def test_forward_and_gradients(shape, dtype, fused) -> None:
    batch, steps, dim = shape
    gate, value, h0 = _inputs(batch, steps, dim, dtype, 7 * steps + dim, fused)
    gen = torch.Generator().manual_seed(5)
    reset = (torch.rand(batch, steps, generator=gen) < 0.05).cuda() if steps % 2 else None
    grad = torch.randn(batch, steps, dim, generator=gen).to(dtype).cuda()
    grad_last = torch.randn(batch, dim, generator=gen).cuda()
    gate, value, h0 = (t.detach().requires_grad_() for t in (gate, value, h0))
    h, last = tropnn_b200.gated_recurrence_b200(gate, value, h0, reset=reset)
    assert h.dtype == dtype and last.dtype == torch.float32
    df, dx, dh0 = torch.autograd.grad([h, last], [gate, value, h0], [grad, grad_last])
    want = _reference(gate, value, h0, reset, grad, grad_last)
    _close(h, want[0], dtype)
    _close(last, want[1], torch.float32)
    _close(df, want[2], dtype)
    _close(dx, want[3], dtype)
    _close(dh0, want[4], torch.float32)


@pytest.mark.parametrize("which", ["h", "last"])
def test_one_output_alone(which) -> None:
    gate, value, _ = _inputs(2, 200, 70, torch.float32, 3)
    gate, value = gate.requires_grad_(), value.requires_grad_()
    h, last = tropnn_b200.gated_recurrence_b200(gate, value)
    out = h if which == "h" else last
    grad = torch.randn(out.shape, generator=torch.Generator().manual_seed(1)).cuda()
    df, dx = torch.autograd.grad(out, [gate, value], grad)
    full = grad if which == "h" else torch.zeros_like(h)
    want = _reference(gate, value, None, None, full, None if which == "h" else grad)
    _close(df, want[2], torch.float32)
    _close(dx, want[3], torch.float32)


def test_gradient_against_differences() -> None:
    """Along one direction: the loss is linear in h, and f32 rounding of a sum of some 10^4 terms of
    size 1 (2^-24 each, adding up like a walk: 1e-5) over a step of 1e-2 leaves 1e-3; the
    difference's own error is of its square."""
    gate, value, h0 = _inputs(2, 150, 40, torch.float32, 11)
    gen = torch.Generator().manual_seed(2)
    weight = torch.randn(2, 150, 40, generator=gen).cuda()
    way = [torch.randn(t.shape, generator=gen).cuda() for t in (gate, value, h0)]
    leaves = [t.clone().requires_grad_() for t in (gate, value, h0)]
    loss = (tropnn_b200.gated_recurrence_b200(*leaves)[0].double() * weight).sum()
    slope = sum((g.double() * w).sum() for g, w in zip(torch.autograd.grad(loss, leaves), way))

    def at(eps):
        moved = [t + eps * w for t, w in zip((gate, value, h0), way)]
        return (tropnn_b200.gated_recurrence_b200(*moved)[0].double() * weight).sum()

    eps = 1e-2
    numeric = (at(eps) - at(-eps)) / (2 * eps)
    assert abs(float(numeric - slope)) <= 2e-3 * (1 + abs(float(slope)))


def test_broadcast_state_gets_the_summed_gradient() -> None:
    gate, value, _ = _inputs(6, 33, 48, torch.float32, 4)
    h0 = torch.randn(48, device="cuda", requires_grad=True)
    h, _ = tropnn_b200.gated_recurrence_b200(gate, value, h0.expand(6, 48))
    (got,) = torch.autograd.grad(h.sum(), h0)  # an expanded upstream gradient too
    want = _reference(gate, value, h0.detach().expand(6, 48), None, torch.ones_like(h))[4].sum(0)
    _close(got, want, torch.float32)


def test_strided_views_and_odd_offsets() -> None:
    """Time-major storage, a step stride of two tokens, a start that is not aligned for pairs."""
    base = torch.randn(70, 3, 2, 41, generator=torch.Generator().manual_seed(9)).cuda()
    for dtype in DTYPES:
        b = base.to(dtype)
        gate = b[:, :, 0, 1:].transpose(0, 1)[:, ::2]
        value = b[:, :, 1, :-1].transpose(0, 1)[:, 1::2]
        h, last = tropnn_b200.gated_recurrence_b200(gate, value)
        want = _reference(gate, value, None, None)
        _close(h, want[0], dtype)
        _close(last, want[1], torch.float32)
    gate = base[..., 0, :].permute(1, 2, 0)  # no unit stride: copied
    h, _ = tropnn_b200.gated_recurrence_b200(gate, gate)
    _close(h, _reference(gate, gate, None, None)[0], torch.float32)


def test_no_steps_no_rows() -> None:
    empty = torch.empty(2, 0, 8, device="cuda")
    h0 = torch.randn(2, 8, device="cuda", requires_grad=True)
    h, last = tropnn_b200.gated_recurrence_b200(empty, empty, h0)
    assert h.shape == (2, 0, 8) and torch.equal(last, h0)
    assert torch.equal(torch.autograd.grad(last.sum(), h0)[0], torch.ones_like(h0))
    for shape in ((0, 5, 8), (2, 5, 0)):
        t = torch.empty(shape, device="cuda")
        h, last = tropnn_b200.gated_recurrence_b200(t, t)
        assert h.shape == shape and last.shape == (shape[0], shape[2])


def test_saturated_gates() -> None:
    """+inf keeps the state, -inf takes the value, exactly."""
    inf = float("inf")
    gate = torch.tensor([inf, -inf, inf, inf, -inf], device="cuda").view(1, 5, 1).expand(1, 5, 3).contiguous()
    value = torch.randn(1, 5, 3, generator=torch.Generator().manual_seed(0)).cuda() * 1e-3
    h0 = torch.full((1, 3), 1e6, device="cuda")
    h, last = tropnn_b200.gated_recurrence_b200(gate, value, h0)
    want = torch.stack([h0, value[:, 1], value[:, 1], value[:, 1], value[:, 4]], dim=1)
    assert torch.equal(h, want) and torch.equal(last, value[:, 4])


def test_long_memory() -> None:
    """a = sigmoid(9), 1 - a = 1.2e-4: some 8000 tokens of memory. The f32 next to a is up to 2^-25 off,
    which a constant gate adds up to 2^-25 / (1 - a) = 2.4e-4 of the state, and rounding the products
    of a's as much again."""
    value = torch.ones(1, 20000, 2, device="cuda")
    value[..., 1] = torch.randn(20000, generator=torch.Generator().manual_seed(1)).cuda() + 1.0
    gate = torch.full_like(value, 9.0)
    h, _ = tropnn_b200.gated_recurrence_b200(gate, value)
    want, _ = _reference(gate, value, None, None)
    assert float((h.double().cpu() - want).abs().max() / want.abs().max()) <= 5e-4


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
@pytest.mark.parametrize("start", [1, 63, 64, 100, 128, 300])
def test_reset_drops_whatever_came_before(start, poison) -> None:
    gate, value, h0 = _inputs(1, 400, 66, torch.float32, 6)
    value[:, :start] = poison
    h0[:] = poison
    reset = torch.zeros(1, 400, dtype=torch.bool, device="cuda")
    reset[0, start] = True
    h, last = tropnn_b200.gated_recurrence_b200(gate, value, h0, reset=reset)
    tail_h, tail_last = _reference(gate[:, start:], value[:, start:], None, None)
    _close(h[:, start:], tail_h, torch.float32)
    _close(last, tail_last, torch.float32)


STRETCHES = [  # one tile a CTA and clusters of tiles, segments in a cluster and in two launches; TMA, pairs, single channels
    (1, 400, 66, torch.float32),
    (2, 1100, 128, torch.bfloat16),
    (40, 300, 256, torch.float16),
    (3, 700, 51, torch.float16),
    (1, 6000, 96, torch.float32),
    (2, 20011, 24, torch.float16),
    (1, 20011, 21, torch.float32),
]


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize(("batch", "steps", "dim", "dtype"), STRETCHES)
def test_resets_that_are_all_false_hide_nothing(batch, steps, dim, dtype, poison) -> None:
    """A value that is not finite stays one for all later tokens, and a gradient for all earlier ones, also
    where the gates between multiply to less than f32 holds: reset false throughout is no reset."""
    gen = torch.Generator().manual_seed(steps)
    gate = torch.randn(batch, steps, dim, generator=gen).to(dtype).cuda()
    value = torch.randn(batch, steps, dim, generator=gen).to(dtype).cuda()
    grad = torch.randn(batch, steps, dim, generator=gen).to(dtype).cuda()
    value[:, 0] = poison
    grad[:, -1, ::2] = poison
    runs = []
    for reset in (None, torch.zeros(batch, steps, dtype=torch.bool, device="cuda")):
        leaves = [t.detach().requires_grad_() for t in (gate, value)]
        h, last = tropnn_b200.gated_recurrence_b200(*leaves, reset=reset)
        runs.append((h, last, *torch.autograd.grad(h, leaves, grad)))
    assert not bool(runs[0][1].isfinite().any()) and not bool(runs[0][3][:, 0, ::2].isfinite().any())
    for got, want in zip(runs[1], runs[0]):
        assert torch.equal(got.isfinite(), want.isfinite())
        assert torch.equal(got[want.isfinite()], want[want.isfinite()])


@pytest.mark.parametrize(("batch", "steps", "dim", "dtype"), STRETCHES)
@pytest.mark.parametrize("part", [0.1, 0.5, 0.97])
def test_reset_drops_a_nan_of_a_gate(batch, steps, dim, dtype, part) -> None:
    """Gates that are NaN on one side of a reset leave states and gradients of the other side alone."""
    gate, value, h0 = _inputs(batch, steps, dim, dtype, 9)
    start = int(part * steps)
    reset = torch.zeros(batch, steps, dtype=torch.bool, device="cuda")
    reset[:, start] = True
    grad = torch.randn(batch, steps, dim, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    none = torch.zeros(batch, dim, device="cuda")
    for bad, good in ((slice(0, start), slice(start, steps)), (slice(start, steps), slice(0, start))):
        poisoned = gate.clone()
        poisoned[:, bad] = float("nan")
        leaves = [t.detach().requires_grad_() for t in (poisoned, value, h0)]
        h, last = tropnn_b200.gated_recurrence_b200(*leaves, reset=reset)
        got = (h, *torch.autograd.grad([h, last], leaves, [grad, none]))
        first = h0 if good.start == 0 else None
        want = _reference(gate[:, good], value[:, good], first, None, grad[:, good])
        for mine, ref in zip(got[:3], (want[0], want[2], want[3])):
            _close(mine[:, good], ref, dtype)
        if good.start == 0:
            _close(got[3], want[4], torch.float32)
        else:
            _close(last, want[1], torch.float32)


def test_reset_at_the_first_and_last_token_and_everywhere() -> None:
    gate, value, h0 = _inputs(3, 70, 64, torch.float32, 8)
    reset = torch.zeros(3, 70, dtype=torch.uint8, device="cuda")
    reset[0, 0] = reset[1, 69] = 1
    reset[2] = 7  # any value but zero
    leaves = [t.requires_grad_() for t in (gate, value, h0)]
    h, last = tropnn_b200.gated_recurrence_b200(*leaves, reset=reset)
    grads = torch.autograd.grad([h, last], leaves, [torch.ones_like(h), torch.ones_like(last)])
    want = _reference(gate, value, h0, reset, torch.ones_like(h), torch.ones_like(last))
    for got, ref in zip((h, last, *grads), want):
        _close(got, ref, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("batch", "dim"), [(1, 1), (3, 77), (8, 1024), (130, 257)])
def test_steps_continue_a_prefill(batch, dim, dtype) -> None:
    gate, value, h0 = _inputs(batch, 6, dim, dtype, dim, fused=True)
    reset = (torch.rand(batch, 6, generator=torch.Generator().manual_seed(2)) < 0.3).cuda()
    want, want_last = _reference(gate, value, h0, reset)
    _, state = tropnn_b200.gated_recurrence_b200(gate[:, :3], value[:, :3], h0, reset=reset[:, :3])
    room = torch.full((batch, dim + 5), float("nan"), device="cuda")  # a state with rows further apart
    room[:, :dim] = state
    state = room[:, :dim]
    for t in range(3, 6):
        h = tropnn_b200.gated_recurrence_step_b200(gate[:, t], value[:, t], state, reset=reset[:, t])
        _close(h, want[:, t], dtype)
    _close(state, want_last, torch.float32)
    assert bool(room[:, dim:].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_do_not_depend_on_alignment(dtype) -> None:
    """The same rows where four channels lie on one boundary and where a row or a pointer does not."""
    gate, value, h0 = _inputs(70, 1, 260, dtype, 15)
    gate, value = gate[:, 0], value[:, 0]
    reset = (torch.rand(70, generator=torch.Generator().manual_seed(3)) < 0.3).cuda()
    want, want_state = _reference(gate[:, None], value[:, None], h0, reset[:, None])

    def placed(t, pad, offset):
        room = torch.full((t.shape[0] * (t.shape[1] + pad) + offset,), float("nan"), device="cuda", dtype=t.dtype)
        view = room[offset:].view(t.shape[0], -1)[:, : t.shape[1]]
        return view.copy_(t)

    results = []
    for pads in ((0, 0, 0), (4, 8, 12), (1, 0, 0), (0, 3, 0), (0, 0, 2)):
        for offsets in ((0, 0, 0), (4, 4, 4), (1, 0, 0), (0, 2, 0), (0, 0, 3)):
            g, x, s = (placed(t, pad, offset) for t, pad, offset in zip((gate, value, h0), pads, offsets))
            h = tropnn_b200.gated_recurrence_step_b200(g, x, s, reset=reset)
            _close(h, want[:, 0], dtype)
            _close(s, want_state, torch.float32)
            results.append((h, s.clone()))
    for h, s in results[1:]:
        assert torch.equal(h, results[0][0]) and torch.equal(s, results[0][1])


def test_runs_are_bitwise_equal_and_do_not_depend_on_the_batch() -> None:
    gate, value, h0 = _inputs(5, 777, 130, torch.bfloat16, 12)
    runs = []
    for rows in (slice(None), slice(None), slice(2, 3)):
        leaves = [t[rows].detach().requires_grad_() for t in (gate, value, h0)]
        h, last = tropnn_b200.gated_recurrence_b200(*leaves)
        runs.append((h, last, *torch.autograd.grad(h.float().sum() + last.sum(), leaves)))
    assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1]))
    assert all(torch.equal(a[2:3], b) for a, b in zip(runs[0], runs[2]))


def test_side_stream_and_two_backwards() -> None:
    gate, value, h0 = _inputs(2, 500, 96, torch.float16, 13)
    leaves = [t.requires_grad_() for t in (gate, value, h0)]
    want = _reference(gate, value, h0, None)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        h, last = tropnn_b200.gated_recurrence_b200(*leaves)
        first = torch.autograd.grad(h.sum(), leaves, retain_graph=True)
        again = torch.autograd.grad(h.sum(), leaves)
    torch.cuda.current_stream().wait_stream(stream)
    _close(h, want[0], torch.float16)
    _close(last, want[1], torch.float32)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_offsets_past_32_bits() -> None:
    far = (1 << 31) + 64
    store = torch.zeros(far + 4096, dtype=torch.float16, device="cuda")
    view = store.as_strided((2, 30, 64), (far, 64, 1))
    gate, value, _ = _inputs(2, 30, 64, torch.float16, 14)
    view.copy_(gate)
    h, last = tropnn_b200.gated_recurrence_b200(view, value)
    want = _reference(gate, value, None, None)
    _close(h, want[0], torch.float16)
    _close(last, want[1], torch.float32)


def test_a_step_tells_autograd_that_it_changed_the_state() -> None:
    gate, value, h0 = _inputs(3, 4, 16, torch.float32, 16)
    _, state = tropnn_b200.gated_recurrence_b200(gate, value, h0)
    weight = torch.ones(16, device="cuda", requires_grad=True)
    loss = (weight * state).sum()  # keeps the state for the weight's gradient
    with torch.no_grad():
        tropnn_b200.gated_recurrence_step_b200(gate[:, 0], value[:, 0], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        _, state = tropnn_b200.gated_recurrence_b200(gate, value, h0)
        tropnn_b200.gated_recurrence_step_b200(gate[:, 0], value[:, 0], state)
    with torch.no_grad():
        tropnn_b200.gated_recurrence_step_b200(gate[:, 0], value[:, 0], state)  # of inference mode: as before


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(grad_mode) -> None:
    """A tangent is not lost, which would be a derivative of 0."""
    gate, value, h0 = _inputs(2, 5, 16, torch.float32, 17)
    for place in range(3):
        with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
            args = [gate, value, h0]
            tropnn_b200.gated_recurrence_b200(*args)
            args[place] = torch.autograd.forward_ad.make_dual(args[place], torch.ones_like(args[place]))
            with pytest.raises(NotImplementedError):
                tropnn_b200.gated_recurrence_b200(*args)
            row = [args[0][:, 0], args[1][:, 0], args[2]]
            with pytest.raises(NotImplementedError):
                tropnn_b200.gated_recurrence_step_b200(*row)


def _elsewhere(t):
    """The same numbers with other strides, as a saved-tensor hook may bring them back."""
    room = torch.full((2, *reversed(t.shape)), 0, dtype=t.dtype, device=t.device)
    return room[0].permute(tuple(reversed(range(t.ndim)))).copy_(t.detach())


def test_saved_tensors_may_come_back_with_other_strides() -> None:
    gate, value, h0 = _inputs(2, 90, 48, torch.float32, 18)
    reset = (torch.rand(2, 90, generator=torch.Generator().manual_seed(4)) < 0.1).cuda()
    leaves = [t.requires_grad_() for t in (gate, value, h0)]
    want = torch.autograd.grad(tropnn_b200.gated_recurrence_b200(*leaves, reset=reset)[0].sum(), leaves)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _elsewhere):
        h, _ = tropnn_b200.gated_recurrence_b200(*leaves, reset=reset)
        got = torch.autograd.grad(h.sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_in_a_cuda_graph() -> None:
    """Forward, backward and steps captured once and replayed on other inputs."""
    gate, value, h0 = _inputs(2, 400, 64, torch.bfloat16, 19)
    long_gate, long_value, _ = _inputs(1, 12000, 32, torch.bfloat16, 20)
    leaves = [t.clone().requires_grad_() for t in (gate, value, h0)]
    state = h0.clone()

    def calls():
        h, last = tropnn_b200.gated_recurrence_b200(*leaves)
        grads = torch.autograd.grad(h, leaves, torch.ones_like(h))
        with torch.no_grad():
            far, _ = tropnn_b200.gated_recurrence_b200(long_gate, long_value)
            step = tropnn_b200.gated_recurrence_step_b200(leaves[0][:, 0], leaves[1][:, 0], state)
        return [h.detach(), last.detach(), *grads, far, step]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        calls()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    with torch.no_grad():
        for t in leaves:
            t.neg_()
        long_value.neg_()
        state.copy_(h0)
    graph.replay()
    got = [t.clone() for t in out]
    state.copy_(h0)
    assert all(torch.equal(a, b) for a, b in zip(got, calls()))


def test_refusals() -> None:
    op, step = tropnn_b200.gated_recurrence_b200, tropnn_b200.gated_recurrence_step_b200
    t = torch.zeros(2, 3, 4, device="cuda")
    row, state = t[:, 0], torch.zeros(2, 4, device="cuda")
    for call in (
        lambda: op(t, t[:, :2]),
        lambda: op(t[0], t[0]),
        lambda: op(t, t, torch.zeros(3, 4, device="cuda")),
        lambda: op(t, t, reset=torch.zeros(2, 4, dtype=torch.bool, device="cuda")),
        lambda: op(t, t.cpu()),
        lambda: step(t, t, state),
        lambda: step(row, row, state[:1]),
        lambda: step(row, row, state[:1].expand(2, 4)),
        lambda: step(row.requires_grad_(), row, state),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (
        lambda: op(t.detach().double(), t.detach().double()),
        lambda: op(t.detach(), t.detach().half()),
        lambda: op(t, t, reset=torch.zeros(2, 3, device="cuda")),
        lambda: step(row.detach(), row.detach(), state.half()),
    ):
        with pytest.raises(TypeError):
            call()
    leaf = torch.zeros(1, 2, 4, device="cuda", requires_grad=True)
    (first,) = torch.autograd.grad(op(leaf, leaf)[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), leaf)
