"""GPU test of the example that runs the training-step operators together with
Muon: the student's loss falls, and all kernels ran to their end."""
from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_student_learns(cuda_device):
    from muon_fusion_ascend950_b200.capi import capi

    path = Path(__file__).resolve().parent.parent / "examples" / "train_student.py"
    spec = importlib.util.spec_from_file_location("train_student", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    before = capi().train_launch_count()
    losses = example.train(steps=60)
    # a step: 4 residual norms (forward, backward, sums), 2 routings (forward,
    # backward), the loss with its gradient
    assert capi().train_launch_count() - before >= 60 * (4 * 3 + 2 * 2 + 1)
    assert all(math.isfinite(v) for v in losses)
    assert losses[-1] < 0.6 * losses[0], (losses[0], losses[-1])
    assert capi().train_device_status(0) == 0
