"""Fits a small Gaussian scene to images of another one: render, backward,
clipped AdamW step, one view a step.

    python examples/fit_scene.py [--steps 200] [--gaussians 10000]

What a step uses of xsimgs_b200: `spherical_harmonics_fused` and
`ut_gs_render` forward and backward, and `AdamW` over all leaves, with
  * a learning rate for each leaf,
  * the global gradient norm, clipped to `max_norm`; a step whose norm is not
    finite is passed over,
  * row masks: Gaussians that the step's view did not see keep their values
    and moments.
The norm of each leaf is printed now and then.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import xsimgs_b200 as X  # noqa: E402
from xsimgs_b200 import scenes  # noqa: E402

LEARNING_RATES = dict(means=2e-3, quats=2e-3, log_scales=5e-3, logits=2e-2, sh=5e-3)


def render(camera, spec, means, quats, log_scales, logits, sh):
    colors = X.spherical_harmonics_fused(sh, means, camera.t0, 0)
    return X.ut_gs_render(camera, means, log_scales.exp(), torch.nn.functional.normalize(quats, dim=-1),
                          logits.sigmoid(), spec.width, spec.height, colors=colors)


def leaves_of(scene):
    return dict(means=scene.means.clone(), quats=scene.quats.clone(), log_scales=scene.scales.log(),
                logits=torch.logit(scene.opacities.clamp(1e-4, 1 - 1e-4)), sh=scene.sh.clone())


def fit(steps=200, gaussians=10_000, max_norm=1.0, device="cuda:0", log=print, seed=0):
    """Mean squared image error of each step."""
    device = torch.device(device)
    spec = scenes.c1_camera()
    views = [spec] + [scenes.pinhole(spec.width, spec.height, 250.0, 250.0, eye, (0.0, 0.0, 10.0))
                      for eye in ((-2.0, 0.0, 0.0), (2.0, 0.0, 0.0), (0.0, 1.5, 0.0))]
    cameras = [v.make(device) for v in views]
    truth = leaves_of(scenes.c1_scene(gaussians, seed).to(device))
    with torch.no_grad():
        targets = [render(c, v, **truth)[0] for c, v in zip(cameras, views)]
    g = torch.Generator().manual_seed(seed + 1)
    spread = dict(means=0.05, quats=0.1, log_scales=0.3, logits=0.5, sh=0.5)
    leaves = {k: (v + spread[k] * torch.randn(v.shape, generator=g).to(device)).requires_grad_()
              for k, v in truth.items()}
    optimizer = X.AdamW([dict(params=[p], lr=LEARNING_RATES[k]) for k, p in leaves.items()], eps=1e-15,
                        max_norm=max_norm, skip_nonfinite=True)
    losses = []
    for step in range(steps):
        i = step % len(views)
        optimizer.zero_grad(set_to_none=True)
        color, _, _, meta = render(cameras[i], views[i], **leaves)
        loss = (color - targets[i]).square().mean()
        loss.backward()
        seen = (meta["radii"] > 0).all(dim=-1)
        if step % 50 == 0:
            _, each = X.gradient_norm([p.grad for p in leaves.values()], per_tensor=True)
            norms = ", ".join(f"{k} {float(n):.2e}" for k, n in zip(leaves, each))
            log(f"step {step}: loss {float(loss.detach()):.5f}, {int(seen.sum())} of {gaussians} seen, gradient norms: {norms}")
        optimizer.step(row_masks={p: seen for p in leaves.values()})
        losses.append(loss.detach())
    return torch.stack(losses).cpu()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--gaussians", type=int, default=10_000)
    a = ap.parse_args()
    losses = fit(a.steps, a.gaussians)
    k = max(1, min(8, len(losses) // 4))
    print(f"loss {float(losses[:k].mean()):.5f} -> {float(losses[-k:].mean()):.5f}")
