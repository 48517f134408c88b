"""The example that runs the renderer, its backward and the clipped AdamW step
together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_fit_scene_lowers_the_loss(cuda):
    spec = importlib.util.spec_from_file_location("fit_scene", os.path.join(ROOT, "examples", "fit_scene.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    lines = []
    losses = example.fit(steps=120, gaussians=3000, log=lines.append)
    assert torch.isfinite(losses).all() and len(lines) == 3
    assert losses[-8:].mean() < 0.5 * losses[:8].mean()
