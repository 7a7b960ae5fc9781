"""Runs of no rows or tokens: a program whose batch is empty has null tensors in hand."""

from __future__ import annotations

import pytest

from arthip_b200.engine import EngineHarnessError
from arthip_b200.token_ops import AxisRotary, TokenNorm
from test_token_ops_cpu import BASE, fake, fake_lib, refused  # noqa: F401


def test_norm_of_no_rows_takes_null_tensors(fake):  # noqa: F811
    op = TokenNorm(64, post_norm="rms")
    before = fake.fake_launches()
    op.run(0, 0, 0, 0, 0, 0)
    op.run(0, 0, norm_ptr=0)
    op.run(0, BASE, BASE, BASE, BASE, rows_per_gate=7)
    refused("rows", op.run, 0, 0, rows_per_gate=0)
    refused("rows", op.run, -1, 0)
    refused("device 1", op.run, 0, 0, stream=0x1000)
    assert fake.fake_launches() - before <= 3


def test_rope_of_no_tokens_takes_null_tensors(fake):  # noqa: F811
    op = AxisRotary(64, [64])
    op.run(0, 0, 0, 2, 0, 0, 2, 0)
    op.run(0, BASE, BASE, 2, BASE + 4096, 0, 2, 0)
    refused("tokens", op.run, -1, 0, 0, 2)
    refused("heads", op.run, 0, BASE, BASE, 0)
    with pytest.raises(EngineHarnessError):
        op.run(1, 0, 0, 2)
