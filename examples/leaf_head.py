"""A softmax head on the leaves of a boosted model.

A boosted model is trained first; each row's leaf in each tree is then a token,
and a small head learns a vector for every leaf.  One training step is

    h = embed(table, leaves)            summed over the trees
    d = dropout(h, p, seed)
    logits = d @ W.T + b                softmax cross entropy
    ... backwards: dropout with the same seed, then embed_grad

and ``answer`` draws classes from the logits.

    python examples/leaf_head.py        # needs a CUDA device
"""
import ctypes as C
import pathlib
import sys

import numpy as np
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))
import ferrisboost_b200 as fb  # noqa: E402
from ferrisboost_b200 import ops  # noqa: E402


class LeafTokens:
    """A model's leaves as tokens: node i of tree t is token first[t] + i."""

    def __init__(self, model: fb.Model):
        self.model = model
        sizes = [len(model.tree(t)["left"]) for t in range(model.num_trees)]
        self.first = torch.tensor(np.concatenate([[0], np.cumsum(sizes)[:-1]]), dtype=torch.int32, device="cuda")
        self.vocab = int(sum(sizes))

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """Tokens (n x trees, int32) of rows that are on the GPU (n x features, float32)."""
        x = x.contiguous()
        if x.dtype != torch.float32 or x.dim() != 2 or x.shape[1] != self.model.n_features:
            raise ValueError(f"rows must be float32 with {self.model.n_features} features, got {x.dtype} {tuple(x.shape)}")
        leaf = torch.empty((x.shape[0], len(self.first)), device=x.device)
        stream = torch.cuda.current_stream(x.device).cuda_stream
        if fb.lib().fbgpu_explain_device(self.model.device_handle(x.get_device()), 0, C.c_void_p(x.data_ptr()),
                                         x.shape[0], C.c_void_p(leaf.data_ptr()), C.c_void_p(stream)):
            raise RuntimeError((fb.lib().fbgpu_last_error(None) or b"").decode())
        return leaf.to(torch.int32) + self.first


class LeafHead:
    """A vector for each leaf and a softmax over their sum, trained with Adagrad."""

    def __init__(self, vocab: int, trees: int, classes: int, dim: int = 32, dropout: float = 0.1, lr: float = 0.1,
                 seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.scale, self.p, self.lr, self.seed, self.steps = trees ** -0.5, dropout, lr, seed, 0
        self.table = 0.1 * torch.randn((vocab, dim), generator=gen, device="cuda")
        self.weight = dim ** -0.5 * torch.randn((classes, dim), generator=gen, device="cuda")
        self.bias = torch.zeros(classes, device="cuda")
        self.squares = [torch.zeros_like(v) for v in (self.table, self.weight, self.bias)]

    def gradients(self, leaves: torch.Tensor, labels: torch.Tensor, seed: int):
        """(loss, gradients of table, weight and bias) of the mean cross entropy under the dropout of `seed`."""
        h = ops.embed(self.table, leaves, scale=self.scale)
        d = ops.dropout(h, self.p, seed)
        log_p = torch.log_softmax(d @ self.weight.T + self.bias, dim=1)
        loss = -log_p.gather(1, labels[:, None]).mean()
        g = log_p.exp()
        g.scatter_add_(1, labels[:, None], torch.full_like(g[:, :1], -1.0))
        g /= len(labels)
        g_h = ops.dropout(g @ self.weight, self.p, seed, out=h)  # h is no longer needed
        g_table = ops.embed_grad(g_h, leaves, len(self.table), scale=self.scale)
        return loss, (g_table, g.T @ d, g.sum(0))

    def step(self, leaves: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        """One training step on a batch; returns its loss, on the GPU."""
        self.steps += 1
        loss, grads = self.gradients(leaves, labels, self.seed + self.steps)
        for v, s, g in zip((self.table, self.weight, self.bias), self.squares, grads):
            s.addcmul_(g, g)
            v.addcdiv_(g, s.sqrt().add_(1e-8), value=-self.lr)
        return loss

    def logits(self, leaves: torch.Tensor) -> torch.Tensor:
        return ops.embed(self.table, leaves, scale=self.scale) @ self.weight.T + self.bias

    def answer(self, leaves: torch.Tensor, u: torch.Tensor, **limits):
        """A class drawn for each row, and its probability (see ops.sample)."""
        return ops.sample(self.logits(leaves), u, **limits)


def data(n: int, classes: int, seed: int):
    """Rows in rings and stripes that a linear model cannot tell apart."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, 8), dtype=np.float32)
    z = np.floor(2.0 * np.hypot(x[:, 0], x[:, 1]) + np.abs(x[:, 2])).astype(np.int64) + (x[:, 3] > 0)
    return x, (z % classes).astype(np.float32)


def main(n: int = 200_000, classes: int = 6, rounds: int = 20, epochs: int = 3, batch: int = 8192) -> dict:
    x, y = data(n, classes, 1)
    model = fb.train({"objective": "multi:softprob", "num_class": classes, "max_depth": 6, "eta": 0.3}, x, label=y,
                     num_boost_round=rounds)
    tokens = LeafTokens(model)
    leaves, labels = tokens(torch.from_numpy(x).cuda()), torch.from_numpy(y).cuda().long()
    head = LeafHead(tokens.vocab, leaves.shape[1], classes)
    losses = []
    for _ in range(epochs):
        for a in range(0, n, batch):
            losses.append(head.step(leaves[a:a + batch], labels[a:a + batch]))
    xt, yt = data(20_000, classes, 2)
    held = tokens(torch.from_numpy(xt).cuda())
    u = torch.rand(len(xt), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    truth = torch.from_numpy(yt).cuda().int()
    best, _ = head.answer(held, u, temperature=0.0)
    drawn, share = head.answer(held, u, temperature=0.7, top_k=3, top_p=0.95)
    boosted = torch.from_numpy(model.predict(xt).argmax(1).astype(np.int32)).cuda()
    return {"first_loss": float(torch.stack(losses[:10]).mean()), "last_loss": float(torch.stack(losses[-10:]).mean()),
            "boosted": float((boosted == truth).float().mean()), "best": float((best == truth).float().mean()),
            "drawn": float((drawn == truth).float().mean()), "share": float(share.mean())}


if __name__ == "__main__":
    for name, value in main().items():
        print(f"{name:12s} {value:.4f}")
