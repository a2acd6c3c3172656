"""The AdamW plan's host logic, on the CPU: what makes a plan stale."""

from __future__ import annotations

import pytest
import torch

from resihp_megatron_amd import kernels as K


def _plan(params):
    """A plan's record of its parameters, without the image (which needs a GPU)."""
    plan = object.__new__(K.AdamWPlan)
    plan.params = list(params)
    plan.shapes, plan.strides = [p.shape for p in params], [p.stride() for p in params]
    plan.dtypes, plan.ptrs = [p.dtype for p in params], [p.data_ptr() for p in params]
    return plan


@pytest.mark.parametrize("change", ["dtype", "shape", "strides", "address"])
def test_a_parameter_that_changed_makes_its_plan_stale(change):
    """The type among them: at the same address, with the same shape and strides, the kernel would read and write
    elements of another size."""
    buf = torch.zeros(64 * 64 * 2)
    square = lambda t: t[:64 * 64].view(64, 64)  # noqa: E731
    p, q = torch.nn.Parameter(square(buf)), torch.nn.Parameter(torch.zeros(5))
    plan = _plan([q, p])
    assert not plan.moved()
    p.data = {"dtype": square(buf.view(torch.bfloat16)), "shape": buf[:64 * 32].view(32, 64), "strides": square(buf).t(),
              "address": square(buf).clone()}[change]
    assert plan.moved()
    p.data = square(buf)
    assert not plan.moved()
