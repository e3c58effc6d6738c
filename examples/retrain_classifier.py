"""Retraining a small network for an approximate multiplier: table convolutions, an exact dense head, its cross entropy and AdamW.

The convolutions multiply through a truth table in the forward pass and have the exact convolution's gradient, so that the
weights learn to live with the multiplier; the end of the network is exact.  Data are synthetic: noisy images of ten patterns.
With --groups the convolutions are followed by group norm with its activation, with --dropout the features before the head are dropped;
--answer-8bit asks the trained network with its dense layers in 8-bit floating point.

  python examples/retrain_classifier.py --steps 100
  python examples/retrain_classifier.py --steps 100 --groups 8 --dropout 0.1 --answer-8bit
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import tf_approximate_b200 as ax  # noqa: E402


class Classifier(torch.nn.Module):
    def __init__(self, table, classes=10, width=16, groups=0, dropout=0.0):
        super().__init__()
        conv = dict(kernel_size=3, padding="same", activation=None if groups else torch.relu, mul_map_file=table)
        layers = []
        for channels, filters, strides in ((3, width, 1), (width, 2 * width, 2), (2 * width, 4 * width, 2)):
            layers.append(ax.FakeApproxConv2D(channels, filters, strides=strides, **conv))
            if groups:
                layers.append(ax.GroupNorm(filters, groups, activation="silu"))
        self.features = torch.nn.Sequential(*layers)
        self.hidden = ax.Dense(4 * width, 4 * width, activation="gelu")
        self.dropout = ax.Dropout(dropout, seed=1) if dropout else torch.nn.Identity()
        self.head = ax.Dense(4 * width, classes)

    def embed(self, images):
        pooled = self.features(images).mean((1, 2))
        return self.dropout(self.hidden(pooled, residual=pooled))

    def in_8bit(self):
        """The network as it answers, its dense layers in 8-bit floating point."""
        self.hidden, self.head = ax.Dense8bit(self.hidden), ax.Dense8bit(self.head)
        return self.eval()

    def loss(self, images, labels):
        return self.head.cross_entropy(self.embed(images), labels)

    def forward(self, images):
        return self.head(self.embed(images))


def batches(seed, batch, hw, classes, device):
    g = torch.Generator(device=device).manual_seed(seed)
    patterns = torch.rand(classes, hw, hw, 3, device=device, generator=g) * 2 - 1
    while True:
        labels = torch.randint(classes, (batch,), device=device, generator=g)
        noise = torch.randn(batch, hw, hw, 3, device=device, generator=g)
        yield (patterns[labels] + 0.5 * noise).clamp(-2, 2), labels


def train(steps=100, batch=256, hw=16, classes=10, state_bits=8, lr=3e-3, table=None, device="cuda", groups=0, dropout=0.0, answer_8bit=False):
    """(losses of the steps, share of a fresh batch that is classified right)"""
    torch.manual_seed(0)
    table = ax.Table(array=ax.noisy_table(3001)) if table is None else table
    net = Classifier(table, classes, groups=groups, dropout=dropout).to(device)
    weights, rest = [p for p in net.parameters() if p.dim() > 1], [p for p in net.parameters() if p.dim() == 1]
    optimizer = ax.AdamW([{"params": weights}, {"params": rest, "weight_decay": 0.0}], lr=lr, state_bits=state_bits)
    data, losses = batches(1, batch, hw, classes, device), []
    for _ in range(steps):
        images, labels = next(data)
        loss = net.loss(images, labels)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    net = net.in_8bit() if answer_8bit else net.eval()
    with torch.no_grad():
        images, labels = next(data)
        right = (net(images).argmax(1) == labels).float().mean()
    return torch.stack(losses).tolist(), float(right)


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--batch", type=int, default=256)
    parser.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    parser.add_argument("--groups", type=int, default=0)
    parser.add_argument("--dropout", type=float, default=0.0)
    parser.add_argument("--answer-8bit", action="store_true")
    args = parser.parse_args()
    losses, right = train(args.steps, args.batch, state_bits=args.state_bits, groups=args.groups, dropout=args.dropout, answer_8bit=args.answer_8bit)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print("step %4d  loss %.4f" % (i, losses[i]))
    print("after %d steps: loss %.4f, %.1f %% of a fresh batch right" % (len(losses), losses[-1], 100 * right))
