"""Host side of the token operators that needs no GPU: CPU tensors and bad calls are refused."""

from __future__ import annotations

import re

import pytest
import torch

import tropnn_b200
from tropnn_b200 import _native as nat
from tropnn_b200 import build as b200_build


@pytest.fixture(scope="module")
def lib():
    b200_build.build()
    return nat.load()


def test_cpu_tensors_are_refused() -> None:
    x, at = torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int64)
    for call in (
        lambda: tropnn_b200.gated_recurrence_b200(x[None], x[None]),
        lambda: tropnn_b200.gated_recurrence_step_b200(x, x, x.clone()),
        lambda: tropnn_b200.distill_loss_b200(x, torch.zeros(2, 3), at),
        lambda: tropnn_b200.distill_loss_grad_b200(x, torch.zeros(2, 3), at),
        lambda: tropnn_b200.sample_tokens_b200(x, torch.zeros(2)),
    ):
        with pytest.raises(ValueError, match="requires CUDA tensors"):
            call()


def test_saved_states_are_one_in_8(lib) -> None:
    size = lib.tropnn_b200_recurrence_saved_size
    assert size(2, 8, 10) == 2 * 1 * 10 * 4
    assert size(2, 9, 10) == 2 * 2 * 10 * 4
    assert size(0, 64, 10) == size(2, 0, 10) == size(2, 64, 0) == size(-1, 64, 10) == 0


def test_c_entries_refuse_before_any_device_work(lib) -> None:
    """Statuses and messages of calls that are wrong by their numbers alone; no pointer is read."""
    null = None

    def recurrence(dtype=nat.F32, batch=1, steps=1, dim=4):
        return lib.tropnn_b200_recurrence_forward(null, 0, 0, null, 0, 0, dtype, null, null, batch, steps, dim, null, null,
                                                  null, 0, null, 0, null)

    def distill(dtype=nat.F32, rows=1, vocab=8, top=2, index=nat.I64, temperature=1.0, weight=0.0):
        return lib.tropnn_b200_distill_loss(null, dtype, rows, 1, vocab, 0, vocab, null, nat.F32, null, index, top, null,
                                            -100, temperature, weight, null, null, null)

    def sample(dtype=nat.F32, rows=1, vocab=8):
        return lib.tropnn_b200_sample_tokens(null, dtype, rows, 1, vocab, 0, vocab, null, null, 1.0, null, nat.I64, 0, null,
                                             1.0, null, 0.0, null, null)

    for status, kind, text in (
        (lambda: recurrence(dtype=nat.I64), nat.ERR_DTYPE, "not f32/f16/bf16"),
        (lambda: recurrence(steps=-1), nat.ERR_INVALID, "bad sizes"),
        (lambda: recurrence(), nat.ERR_INVALID, "null pointer"),
        (lambda: distill(dtype=nat.U8), nat.ERR_DTYPE, "not f32/f16/bf16"),
        (lambda: distill(index=nat.I16), nat.ERR_DTYPE, "not i32/i64"),
        (lambda: distill(vocab=0), nat.ERR_INVALID, "bad sizes"),
        (lambda: distill(top=1025), nat.ERR_INVALID, "1024"),
        (lambda: distill(temperature=0.0), nat.ERR_INVALID, "temperature"),
        (lambda: distill(weight=0.5), nat.ERR_INVALID, "without labels"),
        (lambda: distill(), nat.ERR_INVALID, "null pointer"),
        (lambda: sample(dtype=nat.I64), nat.ERR_DTYPE, "not f32/f16/bf16"),
        (lambda: sample(vocab=1 << 31), nat.ERR_INVALID, "bad sizes"),
        (lambda: sample(), nat.ERR_INVALID, "null pointer"),
    ):
        assert status() == kind
        assert text in nat.last_error()
    assert recurrence(batch=0) == distill(rows=0) == sample(rows=0) == nat.OK


def test_no_kernel_ignores_that_a_wait_ran_out() -> None:
    """Each bounded wait for a copy says whether it arrived; a kernel that went on would leave copies on their
    way into shared memory that is not its own any more."""
    ignored = re.compile(r"^\s*(if( constexpr)? \([^()]*\)\s*)?(sm100::)?mbar_wait(_sleep)?\(")
    sources = sorted(b200_build.CSRC_DIR.glob("*.cu"))
    assert sources
    for path in sources:
        for number, line in enumerate(path.read_text().splitlines(), 1):
            assert not ignored.match(line), f"{path.name}:{number}"


def test_sizes_whose_product_overflows_are_refused(lib) -> None:
    for batch, dim in ((1 << 61, 64), (1 << 40, 1 << 40), (1, 1 << 62)):
        status = lib.tropnn_b200_recurrence_step(16, dim, 16, dim, nat.F32, None, batch, dim, 16, dim, 16, None)
        assert status != 0 and "too large" in nat.last_error()
        status = lib.tropnn_b200_recurrence_forward(16, dim, dim, 16, dim, dim, nat.F32, None, None, batch, 1, dim, 16, 16,
                                                    None, 0, None, 0, None)
        assert status != 0 and "too large" in nat.last_error()
    for batch, dim in ((1 << 62, 256), (1 << 61, 64), (1, (1 << 63) - 1)):
        assert lib.tropnn_b200_recurrence_workspace_size(batch, 100, dim, nat.F32) == 0
        assert lib.tropnn_b200_recurrence_saved_size(batch, 100, dim) == 0
