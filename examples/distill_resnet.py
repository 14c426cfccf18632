"""Training a DDF ResNet from a larger one: the teacher's top logits as targets, the student's classifier and the
distillation loss through the library's operators.

    python examples/distill_resnet.py [--steps 20] [--batch 64] [--image 160] [--k 20] [--temperature 2]

Images are random and both networks start from random weights: the program shows the calls and prints the loss, which
falls as the student learns its teacher's answers for the batch.  A teacher that is too large to run beside the
student leaves its targets on disk instead: ``top_logits`` reduces 1000 logits an image to k values, k classes and a
number, and ``distill_loss`` takes them as they are.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ddfnet_b200 import distill_loss, linear_act, top_logits  # noqa: E402
from ddfnet_b200.resnet import MODELS  # noqa: E402


def train(steps=20, batch=64, image=160, k=20, temperature=2.0, teacher="ddf_mul_resnet101",
          student="ddf_mul_resnet50", classes=1000, seed=0):
    """Returns the losses of the steps."""
    torch.manual_seed(seed)
    with torch.device("cuda"):
        teacher = MODELS[teacher](num_classes=classes).eval()
        student = MODELS[student](num_classes=classes).train()
        images = torch.randn(batch, 3, image, image)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        features = teacher.features(images)
        # (a random classifier answers nearly the same for every image: spread its logits as a trained one's)
        logits = linear_act(features, teacher.fc.weight, teacher.fc.bias)
        logits = logits - logits.mean(0)
        logits = logits * (3 / logits.float().std())
        targets = top_logits(logits, k, temperature=temperature)
    optimizer = torch.optim.SGD(student.parameters(), lr=0.02, momentum=0.9)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            logits = linear_act(student.features(images), student.fc.weight, student.fc.bias)
            loss = distill_loss(logits, *targets, temperature=temperature)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return [loss.item() for loss in losses]


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("steps", 20), ("batch", 64), ("image", 160), ("k", 20)):
        parser.add_argument("--" + name, type=int, default=default)
    parser.add_argument("--temperature", type=float, default=2.0)
    for step, loss in enumerate(train(**vars(parser.parse_args()))):
        print(f"step {step:3d}  loss {loss:.4f}")
