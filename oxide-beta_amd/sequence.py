"""A recurrent classifier of MNIST images read row by row, and its training: the example of the
sequence layers (no counterpart in the reference, whose one model is convolutional).

An image is a sequence of 28 steps of 28 pixels.  A linear layer widens each row, ``nn.
GatedRecurrentBlock``s carry a state down the image (root-mean-square norm, gated recurrence,
residual add), a last norm and the mean over the rows feed a linear classifier.  ``train`` builds
one training program -- forward, reverse mode, ``nn.Muon`` over the blocks' matrices and AdamW over
the rest -- captures it and replays it per batch, each batch gathered on the device.

    python sequence.py DIRECTORY [EPOCHS]     trains on the IDX files of DIRECTORY
"""

from __future__ import annotations

import sys

import numpy as np

import data
import nn
import tensor as tn

ROWS, COLUMNS, CLASSES = 28, 28, 10


class RowClassifier(nn.Module):
    """[batch, 1, rows, columns] images to [batch, classes] logits."""

    def __init__(self, features=128, depth=2, columns=COLUMNS, classes=CLASSES):
        self.widen = nn.Linear(columns, features)
        self.blocks = [nn.GatedRecurrentBlock(features) for _ in range(depth)]
        self.norm = nn.RMSNorm(features)
        self.classifier = nn.Conv2d(features, classes, 1)

    def children(self):
        return [self.widen, *self.blocks, self.norm, self.classifier]

    def matrices(self):
        """The parameters an orthogonalised update suits: the blocks' matrices, not the layers in
        and out."""
        return [p for b in self.blocks for p in b.parameters()]

    def forward(self, images):
        batch, _, rows, columns = images.shape
        x = self.widen(images.reshape((batch, rows, columns)))
        for block in self.blocks:
            x = block(x)
        x = self.norm(x)
        features = x.shape[2]
        mean = x.reshape((batch, 1, rows, features)).avg_pool2d((rows, 1), (rows, 1))
        logits = self.classifier(mean.reshape((batch, features, 1, 1)))
        return logits.reshape((batch, logits.shape[1]))


def optimizer(model: RowClassifier, learning_rate=0.02, adamw_learning_rate=3e-3) -> nn.Muon:
    return nn.Muon(model.matrices(), nn.AdamW(adamw_learning_rate, 1e-4),
                   learning_rate=learning_rate)


class Training:
    """The captured step of one batch size: write ``images`` and ``labels`` (device buffers) on
    ``stream``, then ``step()``."""

    def __init__(self, model: RowClassifier, batch: int, update=None):
        images, labels = tn.input((batch, 1, ROWS, COLUMNS)), tn.input((batch,))
        logits = model(images)
        loss = logits.cross_entropy(labels)
        self.program = tn.training_program(loss, optimizer(model) if update is None else update)
        self.batch, self.stream = batch, self.program.stream_handle
        self.images, self.labels = self.program.value(images), self.program.value(labels)
        self.logits, self._loss = self.program.value(logits), self.program.value(loss)
        self.program.capture()

    def step(self) -> None:
        self.program.replay()

    def loss(self) -> float:
        """The last step's loss; InvalidShape if a label was not a class index."""
        self.program.check()
        return float(self._loss.host()[0])


class Evaluation:
    """The forward of ``batch`` images with the model's current parameters."""

    def __init__(self, model: RowClassifier, batch: int):
        images = tn.input((batch, 1, ROWS, COLUMNS))
        logits = model(images)
        self.program = tn.forward_program(logits, [images])
        self.batch, self.stream = batch, self.program.stream_handle
        self.images, self.logits = self.program.value(images), self.program.value(logits)

    def classes(self) -> np.ndarray:
        self.program.run()
        return self.logits.host().argmax(1)


def train(model: RowClassifier, images, labels, batch=128, epochs=1, report=print) -> float:
    """Trains on byte images [n, 784] and labels [n]; returns the last batch's loss."""
    split, step = data.DeviceSplit(images, labels, shuffle=True), Training(model, batch)
    loss = float("nan")
    for epoch in range(epochs):
        for k in range(split.batches(batch)):
            split.gather(k, batch, step.images, step.labels, stream=step.stream)
            step.step()
        if split.batches(batch):
            loss = step.loss()
        report(f"epoch {epoch + 1}: loss {loss:.4f}")
    return loss


def accuracy(model: RowClassifier, images, labels, batch=100) -> float:
    """The share of whole batches' images that the model classifies rightly."""
    split, run = data.DeviceSplit(images, labels, shuffle=False), Evaluation(model, batch)
    import torch

    truth = torch.empty(batch, device="cuda")
    right = 0
    for k in range(split.batches(batch)):
        split.gather(k, batch, run.images, truth, stream=run.stream)
        right += int((run.classes() == labels[k * batch:(k + 1) * batch]).sum())
    return right / max(1, split.batches(batch) * batch)


def main(directory: str, epochs: int = 1) -> None:
    mnist, model = data.Mnist.load(directory), RowClassifier()
    train(model, mnist.train_images, mnist.train_labels, epochs=epochs)
    print(f"test accuracy {accuracy(model, mnist.test_images, mnist.test_labels):.4f}")


if __name__ == "__main__":
    main(sys.argv[1], int(sys.argv[2]) if len(sys.argv) > 2 else 1)
