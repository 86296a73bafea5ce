"""8-bit activation checkpoints in the shipped recipe (GPU): what a training step keeps, and that nothing but the gradients' rounding changes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_the_shipped_recipe_keeps_less_between_forward_and_backward():
    """one sample of the BEVDepth4D recipe.  Every 1x1 convolution of the image backbone reads an fp32 map that nothing else keeps: 12 images
    (6 of them with gradients) of 64 x 176 x (64 + 64 + 2 * (256 + 64)) and so on, less 33 / 32 of a byte a value; the layers of the other
    parts come on top of that bound.  The losses are those of the run without checkpoints."""
    from distill_bev_amd.train_step import Trainer, build_model, make_batch, parse_losses
    batch = make_batch(1, np.random.default_rng(7), DEV, n_points=20000)

    def one(option):
        model, cfg = build_model(seed=0, allow_synthetic_teacher=True)
        tr = Trainer(model, cfg, DEV, channels_last=True, activation_checkpoint=option)
        tr.step(batch)                                        # caches, packed weights, the captured adjacent frame
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        losses = tr.detector.forward_train(**batch)
        torch.cuda.synchronize()
        kept = torch.cuda.memory_allocated() - before
        total = parse_losses(losses)
        tr.optimizer.zero_grad(set_to_none=True)
        total.backward()
        grads = {n: p.grad.double().norm().item() for n, p in tr.detector.named_parameters() if p.grad is not None}
        marks = (tr.detector.act8_modules, tr.detector.act8_bias_convs)
        tr.close()
        return kept, float(total.detach()), grads, marks

    kept, _, grads, marks = one(None)
    kept8, _, grads8, marks8 = one("int8")
    assert marks == (0, 0) and marks8 == (34, 13)
    # inputs of the stages' conv1 / conv3, pixels of an image x channels, 6 images with gradients at 256 x 704
    hw = {1: 64 * 176, 2: 32 * 88, 3: 16 * 44, 4: 8 * 22}
    values = 6 * (hw[1] * (64 + 2 * 256 + 3 * 64) + hw[2] * (3 * 512 + 4 * 128) + hw[3] * (5 * 1024 + 6 * 256) + hw[4] * (2 * 2048 + 3 * 512))
    print(f"kept {kept / 2**20:.0f} MiB, with int8 checkpoints {kept8 / 2**20:.0f} MiB; bound on the difference {values * (4 - 33 / 32) / 2**20:.0f} MiB")
    assert kept - kept8 >= 0.9 * values * (4 - 33 / 32)
    assert set(grads) == set(grads8) and all(np.isfinite(v) for v in grads8.values())


def test_first_loss_and_gradients_with_checkpoints_are_close_to_those_without():
    """the same weights and batch, before any step: the forward pass is the same but for the order of a few library sums"""
    from distill_bev_amd.train_step import Trainer, build_model, make_batch, parse_losses
    batch = make_batch(1, np.random.default_rng(8), DEV, n_points=20000)

    def one(option):
        model, cfg = build_model(seed=0, allow_synthetic_teacher=True)
        tr = Trainer(model, cfg, DEV, channels_last=True, activation_checkpoint=option)
        total = parse_losses(tr.detector.forward_train(**batch))
        total.backward()
        out = float(total.detach()), {n: p.grad.double() for n, p in tr.detector.named_parameters() if p.grad is not None}
        tr.close()
        return out

    la, ga = one(None)
    lb, gb = one("int8")
    assert abs(la - lb) <= 1e-4 * abs(la)
    # a kept value is off by 2^-7 of its block's largest at most: the weights' gradients by a few per cent at random signs (data gradients do
    # not see the checkpoints); taken over all of them, so that layers whose gradient is what is left of a cancellation do not count
    num = sum(float((ga[k] - gb[k]).square().sum()) for k in ga) ** 0.5
    den = sum(float(ga[k].square().sum()) for k in ga) ** 0.5
    print(f"gradients differ by {num / den:.2e}")
    assert num < 0.05 * den
