"""One training step from token ids to clipped parameters through the package's
operators, against the same step in 64 bits with torch's elementary ones."""

from __future__ import annotations

import pytest
import torch

import maxsim_amd

from ._training_helpers import rand

pytestmark = pytest.mark.gpu

VOCAB, HIDDEN, DIM, LQ, LD, BATCH = 500, 96, 64, 9, 41, 12


class _Model(torch.nn.Module):
    """A table of tokens and one of positions, layer norm and a projection."""

    def __init__(self, dtype=torch.float32, seed=0):
        super().__init__()
        gen = torch.Generator().manual_seed(seed)
        new = lambda *shape, scale=1.0: torch.nn.Parameter(rand(gen, *shape, scale=scale).to(dtype))
        self.tokens, self.positions = new(VOCAB, HIDDEN), new(64, HIDDEN, scale=0.3)
        self.weight, self.bias = new(HIDDEN), new(HIDDEN, scale=0.1)
        self.project = new(DIM, HIDDEN, scale=HIDDEN ** -0.5)


def _batch(seed):
    gen = torch.Generator().manual_seed(seed)
    ids = lambda n, length: (VOCAB ** torch.rand(n, length, generator=gen, dtype=torch.float64)).long() - 1
    lengths = torch.randint(1, LD + 1, (BATCH,), generator=gen)
    queries, documents = ids(BATCH, LQ), ids(BATCH, LD)
    documents[torch.arange(LD) >= lengths[:, None]] = -7  # padding is never looked up
    return queries.cuda(), documents.cuda(), lengths.cuda()


def _loss(m, batch):
    queries, documents, lengths = batch
    scale = HIDDEN ** 0.5

    def hidden(ids, lens=None):
        at = torch.arange(ids.shape[1], device="cuda").expand(ids.shape)
        x = maxsim_amd.embed_tokens(m.tokens, ids, lens, scale=scale, padding_idx=3)
        x = x + maxsim_amd.embed_tokens(m.positions, at, lens)
        return maxsim_amd.layer_norm(x, m.weight, m.bias) @ m.project.t()

    q = maxsim_amd.normalize_embeddings(hidden(queries))
    d, offsets = maxsim_amd.pack_normalized_documents(hidden(documents, lengths), lengths)
    return maxsim_amd.score_contrastive_cross_entropy(q, d, offsets, temperature=0.3)


def _plain_loss(m, batch):
    queries, documents, lengths = batch
    real = torch.arange(LD, device="cuda") < lengths[:, None]

    def hidden(ids, real=None):
        ids = ids if real is None else torch.where(real, ids, 0)
        table = torch.where(torch.arange(VOCAB, device="cuda")[:, None] == 3, m.tokens.detach(), m.tokens)
        x = table[ids] * HIDDEN ** 0.5
        x = x + m.positions[torch.arange(ids.shape[1], device="cuda")]
        x = x - x.mean(-1, keepdim=True)
        x = x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * m.weight + m.bias
        x = (x.reshape(-1, HIDDEN) @ m.project.t()).view(*ids.shape, DIM)
        return x / x.square().sum(-1, keepdim=True).sqrt()

    q, d = hidden(queries), hidden(documents, real)
    sims = (q.reshape(-1, DIM) @ d.reshape(-1, DIM).t()).view(BATCH, LQ, BATCH, LD)
    scores = sims.masked_fill(~real, -10.0).amax(-1).sum(1)
    return torch.nn.functional.cross_entropy(scores / 0.3, torch.arange(BATCH, device="cuda"))


def test_a_step_from_ids_to_parameters():
    ours, theirs = _Model(), _Model(torch.float64)
    opt = maxsim_amd.AdamW(ours.parameters(), lr=1e-3, weight_decay=0.05, max_norm=0.1)
    plain = torch.optim.AdamW(theirs.parameters(), lr=1e-3, weight_decay=0.05)
    for step in range(3):
        batch = _batch(step)
        opt.zero_grad()
        plain.zero_grad()
        loss, want = _loss(ours, batch), _plain_loss(theirs, batch)
        loss.backward()
        want.backward()
        # each stage is off by a few hundred roundings of fp32 (6e-8) at most, of
        # its largest value
        assert float(loss.detach()) == pytest.approx(float(want.detach()), rel=1e-4)
        for (name, a), b in zip(ours.named_parameters(), theirs.parameters()):
            far = (a.grad.double() - b.grad).abs().max() / b.grad.abs().max()
            assert float(far) < 1e-3, (step, name, float(far))
        assert not ours.tokens.grad[3].any()
        opt.step()
        norm = torch.nn.utils.clip_grad_norm_(theirs.parameters(), 0.1)
        assert float(norm) > 0.1
        assert float(opt.grad_norm) == pytest.approx(float(norm), rel=1e-4)
        plain.step()
        # a step is lr at most in each element, and its sign is the gradient's
        # where that is far from rounding: hold those
        for (name, a), b, g in zip(ours.named_parameters(), theirs.parameters(),
                                   (p.grad for p in theirs.parameters())):
            sure = g.abs() > 1e-2 * g.abs().max()
            far = (a.detach().double() - b.detach())[sure].abs().max()
            assert float(far) < 1e-3 * 1e-1, (step, name, float(far))
        # go on from the same place
        with torch.no_grad():
            for a, b in zip(ours.parameters(), theirs.parameters()):
                b.copy_(a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_steps_in_16_bits(dtype):
    # tables kept in 32 bits and looked up in 16, the head in 16 with masters
    model = _Model()
    table = model.tokens
    head = torch.nn.Parameter((model.project.detach() / 2).to(dtype))
    opt = maxsim_amd.AdamW([table, head], lr=1e-2, state_bits=8, min_8bit_size=1,
                           master_weights=True, max_norm=1.0)
    norms = []
    for step in range(3):
        queries, documents, lengths = _batch(step)
        q = maxsim_amd.embed_tokens(table, queries, dtype=dtype) @ head.t()
        d = maxsim_amd.embed_tokens(table, documents, lengths, dtype=dtype) @ head.t()
        d, offsets = maxsim_amd.pack_normalized_documents(d, lengths)
        loss = maxsim_amd.score_contrastive_cross_entropy(maxsim_amd.normalize_embeddings(q), d, offsets,
                                                          temperature=0.3)
        opt.zero_grad()
        loss.backward()
        assert table.grad.dtype == torch.float32 and head.grad.dtype == dtype
        before = [table.grad.clone(), head.grad.clone()]
        opt.step()
        norms.append(float(opt.grad_norm))
        assert torch.equal(table.grad, before[0]) and torch.equal(head.grad, before[1])
        assert all(bool(torch.isfinite(p).all()) for p in (table, head))
        want = sum(float(g.double().square().sum()) for g in before) ** 0.5
        assert norms[-1] == pytest.approx(want, rel=1e-6)
    assert len(set(norms)) == 3
