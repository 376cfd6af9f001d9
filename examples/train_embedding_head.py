"""Train an embedding head for late interaction on top of a frozen encoder.

What this package covers of such a step, in the order it runs:

    hidden states --layer_norm--> normed --linear (torch)--> projected
      queries:    --normalize_embeddings--> unit token embeddings
      documents:  --pack_normalized_documents--> packed unit embeddings, offsets
    --score_contrastive_cross_entropy--> loss --backward--> gradients --AdamW-->

The hidden states are synthetic: each document is a bag of topics, and its query
repeats some of them.  Half of the coordinates hold the topic, in noise; the
other half hold twice as much of nothing, which the head has to learn to leave
out.  Needs an MI355X.

    python examples/train_embedding_head.py --steps 200 --state-bits 8
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import maxsim_amd  # noqa: E402


class EmbeddingHead(torch.nn.Module):
    """Layer norm and projection of an encoder's hidden states."""

    def __init__(self, hidden: int, dim: int, dtype: torch.dtype):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(hidden, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(hidden, dtype=dtype))
        self.project = torch.nn.Linear(hidden, dim, bias=False, dtype=dtype)

    def forward(self, hidden):
        return self.project(maxsim_amd.layer_norm(hidden, self.weight, self.bias))

    def queries(self, hidden):
        return maxsim_amd.normalize_embeddings(self(hidden))

    def documents(self, hidden, lengths):
        return maxsim_amd.pack_normalized_documents(self(hidden), lengths)


class Batches:
    """Synthetic hidden states of queries and padded documents."""

    def __init__(self, batch, lq, ld, hidden, dtype, seed=0, topics=512):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.batch, self.lq, self.ld, self.hidden, self.dtype = batch, lq, ld, hidden, dtype
        self.topics = self._normal(topics, hidden // 2)

    def _normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def _states(self, pick):
        topic = self.topics[pick] + 0.5 * self._normal(*pick.shape, self.topics.shape[1])
        rest = 2.0 * self._normal(*pick.shape, self.hidden - self.topics.shape[1])
        return torch.cat([topic, rest], dim=-1).to(self.dtype)

    def next(self):
        """Queries [batch, lq, hidden], documents [batch, ld, hidden], lengths."""
        n = self.batch
        lengths = torch.randint(self.ld // 4, self.ld + 1, (n,), generator=self.gen, device="cuda")
        pick = torch.randint(0, self.topics.shape[0], (n, self.ld), generator=self.gen,
                             device="cuda")
        at = (torch.rand(n, self.lq, generator=self.gen, device="cuda") * lengths[:, None]).long()
        return self._states(torch.gather(pick, 1, at)), self._states(pick), lengths


def train(steps=200, batch=64, lq=32, ld=180, hidden=768, dim=128, dtype=torch.bfloat16,
          state_bits=8, lr=2e-3, temperature=0.5, seed=0, report=20):
    """Returns the losses of all steps."""
    torch.manual_seed(seed)
    head = EmbeddingHead(hidden, dim, dtype).cuda()
    optimizer = maxsim_amd.AdamW(head.parameters(), lr=lr, weight_decay=0.01,
                                 state_bits=state_bits, master_weights=dtype != torch.float32)
    data = Batches(batch, lq, ld, hidden, dtype, seed)
    losses = []
    # one GPU per process: backward on this thread saves the hand-over to the
    # engine's, which costs more than the kernels of a small batch
    with torch.autograd.set_multithreading_enabled(False):
        for step in range(steps):
            if step == 1:  # the first one loads kernels and fills allocators
                began = time.perf_counter()
            queries, documents, lengths = data.next()
            q = head.queries(queries)
            d, offsets = head.documents(documents, lengths)
            loss = maxsim_amd.score_contrastive_cross_entropy(q, d, offsets,
                                                              temperature=temperature)
            optimizer.zero_grad()
            loss.backward()
            optimizer.step()
            losses.append(loss.detach())
            if report and step > 0 and (step + 1) % report == 0:
                print(f"step {step + 1:5d}  loss {float(loss.detach()):.4f}  "
                      f"{(time.perf_counter() - began) / step * 1e3:.2f} ms per step", flush=True)
    return torch.stack(losses).tolist()


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--batch", type=int, default=64)
    parser.add_argument("--dtype", choices=("bf16", "f16", "f32"), default="bf16")
    parser.add_argument("--state-bits", type=int, choices=(8, 32), default=8)
    parser.add_argument("--lr", type=float, default=2e-3)
    args = parser.parse_args()
    dtype = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[args.dtype]
    train(args.steps, args.batch, dtype=dtype, state_bits=args.state_bits, lr=args.lr)


if __name__ == "__main__":
    main()
