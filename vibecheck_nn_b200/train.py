"""Train a ReLU classifier with the package's own kernels, then bound it.

``MlpTrainer`` runs the training step -- ``linear.linear_forward`` per layer,
``loss.cross_entropy_grad``, ``linear.linear_backward`` per layer, one
``optim.AdamW`` step -- and hands the network to the bound propagation as a
``gg`` dict.  ``certified`` bounds every class margin over boxes around given
points with CROWN (``ops.ibp_crown_batched``): the points whose margins are all
positive keep their label everywhere in their box.

    python -m vibecheck_nn_b200.train

trains a 5 -> [50] x 3 -> 5 network on points labelled by their nearest of five
centres and prints the loss, the accuracy and the certified fraction.
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib, linear, loss, ops, optim, workloads


class MlpTrainer:
    """fc / ReLU network of (W, b) layers trained with AdamW.

    ``layers`` are arrays as in ``workloads.mlp_params``; weights, activations
    and gradients are ``dtype`` (float32, bfloat16 or float16), the optimiser's
    moments 32 or 8 bits."""

    def __init__(self, layers, device='cuda', dtype=torch.float32, lr=1e-3, weight_decay=0.0,
                 state_bits=32, seed=0):
        put = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.float32, device=device) \
            .to(dtype).contiguous()  # noqa: E731
        self.weights = [put(W) for W, _ in layers]
        self.biases = [put(b) for _, b in layers]
        self.dtype = dtype
        self.opt = optim.AdamW(self.weights + self.biases, lr=lr, weight_decay=weight_decay,
                               state_bits=state_bits, seed=seed)

    def logits(self, x, keep=False):
        """Network outputs (R, C); with ``keep`` also each layer's (input,
        pre-activation) for the backward pass."""
        saved = []
        last = len(self.weights) - 1
        for i, (W, b) in enumerate(zip(self.weights, self.biases)):
            act = 'relu' if i < last else 'none'
            out = linear.linear_forward(x, W, b, act, keep=keep and i < last)
            y, z = out if keep and i < last else (out, None)
            saved.append((x, z))
            x = y
        return (x, saved) if keep else x

    def gradients(self, x, labels):
        """(loss, gradients in the order of the optimiser's parameters)."""
        y, saved = self.logits(x, keep=True)
        value, dy = loss.cross_entropy_grad(y, labels)
        dW, db = [None] * len(saved), [None] * len(saved)
        for i in reversed(range(len(saved))):
            inp, z = saved[i]
            dy, dW[i], db[i] = linear.linear_backward(dy, inp, self.weights[i], z,
                                                      'none' if z is None else 'relu',
                                                      need=(i > 0, True))
        return value, dW + db

    def step(self, x, labels):
        """One training step on points ``x`` (R, n_in) of the network's type;
        returns the loss before it (a device scalar)."""
        value, grads = self.gradients(x, labels)
        self.opt.step(grads)
        return value

    def layers(self):
        """The network as float32 (W, b) arrays; raises ``TimeoutError`` if a
        bounded device wait ran out while it was trained."""
        _lib.fault_check(self.weights[0].device)
        return [(W.float().cpu().numpy(), b.float().cpu().numpy())
                for W, b in zip(self.weights, self.biases)]

    def gg(self):
        """The network as the op dict that the bound propagation takes."""
        return workloads.mlp_gg(self.layers(), self.weights[0].device)


def certified(gg, x, labels, eps):
    """For points ``x`` (R, n_in) float32 with int labels: the lower bounds of
    all margins y_label - y_j over the box of radius ``eps`` around each point
    (R, C; +inf at j = label).  A point is certified when its row is positive."""
    n_out = int(gg['ops'][-1]['W'].shape[0])
    margins = torch.full((x.shape[0], n_out), float('inf'), device=x.device)
    for label in range(n_out):
        rows = torch.nonzero(labels == label)[:, 0]
        if not rows.numel():
            continue
        W_q, b_q = (torch.as_tensor(a, dtype=torch.float32, device=x.device)
                    for a in workloads.margin_rows(n_out, label))
        lb = ops.ibp_crown_batched(x[rows] - eps, x[rows] + eps, gg, (W_q, b_q), x.device)
        others = [j for j in range(n_out) if j != label]
        margins[rows[:, None], torch.tensor(others, device=x.device)] = lb
    return margins


def nearest_centre_data(n, n_in, n_classes, seed=0, device='cuda'):
    """Uniform points of [-1, 1]^n_in labelled by their nearest centre."""
    rng = np.random.default_rng(seed)
    centres = rng.uniform(-1, 1, (n_classes, n_in))
    x = rng.uniform(-1, 1, (n, n_in))
    labels = np.argmin(((x[:, None] - centres[None]) ** 2).sum(-1), 1)
    return (torch.as_tensor(x, dtype=torch.float32, device=device),
            torch.as_tensor(labels, device=device))


def main(steps=400, batch=2048, eps=0.01):
    x, labels = nearest_centre_data(16384, 5, 5)
    layers = workloads.mlp_params((5, 50, 50, 50, 5), np.random.default_rng(0))
    trainer = MlpTrainer(layers, lr=2e-3, weight_decay=1e-3, state_bits=8)
    for step in range(steps):
        a = step * batch % x.shape[0]
        value = trainer.step(x[a:a + batch], labels[a:a + batch])
        if step % 100 == 0 or step == steps - 1:
            print(f'step {step}: loss {float(value):.4f}')
    right = trainer.logits(x).argmax(1) == labels
    safe = (certified(trainer.gg(), x, labels, eps) > 0).all(1)
    print(f'accuracy {float(right.float().mean()):.4f}, certified at radius {eps}: '
          f'{float(safe.float().mean()):.4f}')


if __name__ == '__main__':
    main()
