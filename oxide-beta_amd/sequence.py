"""A recurrent classifier of MNIST images read row by row, and its training: the example of the
sequence layers (no counterpart in the reference, whose one model is convolutional).

An image is a sequence of 28 steps of 28 pixels.  A linear layer widens each row, ``nn.
GatedRecurrentBlock``s carry a state down the image (root-mean-square norm, gated recurrence,
residual add), or with ``block=nn.DeltaRuleBlock`` and ``norm=nn.LayerNorm`` states that a gated
delta rule writes; a last norm and the mean over the rows feed a linear classifier.  ``train``
builds one training program -- forward, reverse mode, ``nn.Muon`` over the blocks' matrices and
AdamW over the rest -- captures it and replays it per batch, each batch gathered on the device.
``train_by_reward`` is told only whether a class that the model drew is the right one, and lowers
the clipped policy loss of its draws.

    python sequence.py DIRECTORY [EPOCHS [delta] [reward]]     trains on the IDX files of DIRECTORY
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

    def __init__(self, features=128, depth=2, columns=COLUMNS, classes=CLASSES,
                 block=nn.GatedRecurrentBlock, norm=nn.RMSNorm):
        self.widen = nn.Linear(columns, features)
        self.blocks = [block(features) for _ in range(depth)]
        self.norm = norm(features)
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


class RewardTraining:
    """The captured step of one batch of drawn classes: write ``images`` on ``stream``, ``draw()``,
    score the draws, then ``step(rewards)``.  Several steps may follow one draw: the clip holds
    them near the policy that drew."""

    def __init__(self, model: RowClassifier, batch: int, update=None, clip=(0.2, 0.2), seed=0):
        images, actions, old, advantages = (tn.input(shape) for shape in (
            (batch, 1, ROWS, COLUMNS), (batch,), (batch,), (batch,)))
        logits = model(images)
        loss = logits.policy_loss(actions, old, advantages, clip=clip)
        self.program = tn.training_program(loss, optimizer(model) if update is None else update)
        self.batch, self.stream = batch, self.program.stream_handle
        self.images, self._loss = self.program.value(images), self.program.value(loss)
        self._rows = [self.program.value(t) for t in (actions, old, advantages)]
        self._model, self._random = Evaluation(model, batch), np.random.default_rng(seed)
        self.program.capture()

    def draw(self) -> np.ndarray:
        """A class per image from the model's current probabilities, kept for the next steps."""
        self._model.images.copy_from(self.images.host())
        self._model.program.run()
        logits = self._model.logits.host().astype(np.float64)
        actions = (logits + self._random.gumbel(size=logits.shape)).argmax(1)
        largest = logits.max(1)
        sums = np.log(np.exp(logits - largest[:, None]).sum(1)) + largest
        self._rows[0].copy_from(actions.astype(np.float32))
        self._rows[1].copy_from((logits[np.arange(self.batch), actions] - sums).astype(np.float32))
        return actions

    def step(self, rewards) -> None:
        """One update; a draw's advantage is its reward above the batch's mean, in deviations."""
        r = np.asarray(rewards, np.float64)
        self._rows[2].copy_from(((r - r.mean()) / (r.std() + 1e-6)).astype(np.float32))
        self.program.replay()

    def loss(self) -> float:
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


def train_by_reward(model: RowClassifier, images, labels, batch=128, epochs=1, steps=2,
                    report=print) -> float:
    """Trains by rewards of 1 for a draw of the right class, ``steps`` updates a draw; returns the
    last batch's mean reward."""
    split = data.DeviceSplit(images, labels, shuffle=True)
    step, reward = RewardTraining(model, batch), float("nan")
    import torch

    truth = torch.empty(batch, device="cuda")
    for epoch in range(epochs):
        for k in range(split.batches(batch)):
            split.gather(k, batch, step.images, truth, stream=step.stream)
            drawn = step.draw()  # waits for the stream: the labels are there, too
            rewards = (drawn == truth.cpu().numpy()).astype(np.float64)
            for _ in range(steps):
                step.step(rewards)
            reward = float(rewards.mean())
        step.program.check()
        report(f"epoch {epoch + 1}: reward {reward:.4f}")
    return reward


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


def main(directory: str, epochs: int = 1, *kinds: str) -> None:
    unknown = set(kinds) - {"delta", "reward"}
    if unknown:
        raise ValueError(f"sequence.py takes delta and reward, not {', '.join(sorted(unknown))}")
    mnist = data.Mnist.load(directory)
    model = (RowClassifier(block=nn.DeltaRuleBlock, norm=nn.LayerNorm) if "delta" in kinds
             else RowClassifier())
    fit = train_by_reward if "reward" in kinds else train
    fit(model, mnist.train_images, mnist.train_labels, epochs=epochs)
    print(f"test accuracy {accuracy(model, mnist.test_images, mnist.test_labels):.4f}")


if __name__ == "__main__":
    main(sys.argv[1], int(sys.argv[2]) if len(sys.argv) > 2 else 1, *sys.argv[3:])
