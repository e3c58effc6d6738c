"""Retraining a small network for an approximate multiplier: table convolutions, an exact dense head, its cross entropy and AdamW.

The convolutions multiply through a truth table in the forward pass and have the exact convolution's gradient, so that the
weights learn to live with the multiplier; the end of the network is exact.  Data are synthetic: noisy images of ten patterns.

  python examples/retrain_classifier.py --steps 100
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import tf_approximate_b200 as ax  # noqa: E402


class Classifier(torch.nn.Module):
    def __init__(self, table, classes=10, width=16):
        super().__init__()
        conv = dict(kernel_size=3, padding="same", activation=torch.relu, mul_map_file=table)
        self.features = torch.nn.Sequential(ax.FakeApproxConv2D(3, width, **conv), ax.FakeApproxConv2D(width, 2 * width, strides=2, **conv),
                                            ax.FakeApproxConv2D(2 * width, 4 * width, strides=2, **conv))
        self.hidden = ax.Dense(4 * width, 4 * width, activation="gelu")
        self.head = ax.Dense(4 * width, classes)

    def embed(self, images):
        pooled = self.features(images).mean((1, 2))
        return self.hidden(pooled, residual=pooled)

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


def train(steps=100, batch=256, hw=16, classes=10, state_bits=8, lr=3e-3, table=None, device="cuda"):
    """(losses of the steps, share of a fresh batch that is classified right)"""
    torch.manual_seed(0)
    table = ax.Table(array=ax.noisy_table(3001)) if table is None else table
    net = Classifier(table, classes).to(device)
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
    net.eval()
    with torch.no_grad():
        images, labels = next(data)
        right = (net(images).argmax(1) == labels).float().mean()
    return torch.stack(losses).tolist(), float(right)


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--batch", type=int, default=256)
    parser.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    args = parser.parse_args()
    losses, right = train(args.steps, args.batch, state_bits=args.state_bits)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print("step %4d  loss %.4f" % (i, losses[i]))
    print("after %d steps: loss %.4f, %.1f %% of a fresh batch right" % (len(losses), losses[-1], 100 * right))
