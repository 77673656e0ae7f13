"""A small example: an integer network learns to tell many classes apart, and a narrower one learns from its best answers.

    python -m niti_amd.distill [--classes 2000] [--steps 400] ...

The data are made up: a class is a random pattern, a sample its pattern with noise.  The teacher (one hidden layer, TiVocabHead) is
trained by cross entropy; the student sees the same samples without their labels, and of the teacher its ``--top`` largest logits.
Every product, loss, gradient and update is the library's."""
from __future__ import annotations

import argparse

import torch

from . import ti_torch
from .ti_torch import TiLinear, TiReLU
from .ti_vocab import TiVocabHead


class Net:
    """features -> hidden -> classes."""

    def __init__(self, features, hidden, classes):
        self.below = [TiLinear(features, hidden), TiReLU()]
        self.head = TiVocabHead(hidden, classes)

    def hidden(self, x):
        for layer in self.below:
            x = layer.forward(x)
        return x

    def step(self, x, grad=None, **what):
        """One training step; the mean loss as a device tensor."""
        loss = self.head.forward(self.hidden(x), **what)
        err = self.head.backward(grad)
        for layer in reversed(self.below):
            err = layer.backward(err)
        return loss.mean()

    def accuracy(self, x, target):
        return (self.head.top_logits(self.hidden(x), 1)[1][:, 0] == target).float().mean()


class Samples:
    def __init__(self, features, classes, noise, seed, device):
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.device, self.noise = device, noise
        self.patterns = torch.randint(-40, 41, (classes, features), generator=self.gen, device=device).float()

    def batch(self, n):
        target = torch.randint(0, len(self.patterns), (n,), generator=self.gen, device=self.device)
        x = self.patterns[target] + self.noise * torch.randn((n, self.patterns.shape[1]), generator=self.gen, device=self.device)
        return (x.round().clamp(-127, 127).to(torch.int8), -5), target


def run(classes=2000, features=256, hidden=512, student=384, batch=256, steps=400, top=16, temperature=1.0, noise=10.0, seed=0, say=print):
    """Returns (teacher's first and last loss, its accuracy, student's first and last loss, its accuracy)."""
    torch.manual_seed(seed)
    device = torch.device(ti_torch.GPU)
    data = Samples(features, classes, noise, seed, device)
    teacher, pupil = Net(features, hidden, classes), Net(features, student, classes)

    def train(name, one):
        first = last = None
        for i in range(steps):
            loss = one()
            if i == 0 or i == steps - 1 or (i + 1) % 100 == 0:      # the only copies to the host
                last = float(loss)
                first = last if first is None else first
                say("%s step %4d  loss %.4f" % (name, i + 1, last))
        return first, last

    def teach():
        x, target = data.batch(batch)
        return teacher.step(x, target=target)

    def learn():
        x, _ = data.batch(batch)
        return pupil.step(x, teacher=teacher.head.top_logits(teacher.hidden(x), top), temperature=temperature)

    t = train("teacher", teach)
    s = train("student", learn)
    x, target = data.batch(4 * batch)
    acc = float(teacher.accuracy(x, target)), float(pupil.accuracy(x, target))
    say("accuracy on new samples: teacher %.1f %%, student %.1f %%" % (100 * acc[0], 100 * acc[1]))
    return t + acc[:1] + s + acc[1:]


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("classes", 2000), ("features", 256), ("hidden", 512), ("student", 384), ("batch", 256), ("steps", 400), ("top", 16), ("seed", 0)):
        p.add_argument("--" + name, type=int, default=value)
    p.add_argument("--temperature", type=float, default=1.0)
    p.add_argument("--noise", type=float, default=10.0)
    run(**vars(p.parse_args(argv)))


if __name__ == "__main__":
    main()
