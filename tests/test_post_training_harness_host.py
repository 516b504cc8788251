"""``Decoder.token_logprobs`` around its decoder: which targets go with which tokens, chunk by chunk (on the CPU, with the decoder, the
projection and the log probabilities replaced by elementary ones)."""
import types

import pytest
import torch

from torchtune_amd import harness
from torchtune_amd.modules import layer_ops

DIM, VOCAB = 6, 11


def _plain(logits, tokens, *, temperature, entropy, top, ignore_index):
    log_p = torch.log_softmax(logits / temperature, -1)
    given = tokens.reshape(*logits.shape[:-1], -1)
    lp = log_p.gather(-1, given).view(tokens.shape)
    alternatives = log_p.sort(-1, descending=True) if top else None
    return layer_ops.TokenLogprobs(lp, -(log_p.exp() * log_p).sum(-1) if entropy else None, *((None, None) if not top else
                                   (alternatives.values[..., :top], alternatives.indices[..., :top])))


@pytest.fixture
def decoder(monkeypatch):
    monkeypatch.setattr(layer_ops, "token_logprobs", _plain)
    g = torch.Generator().manual_seed(0)
    table, weight = torch.randn(VOCAB, DIM, generator=g), torch.randn(VOCAB, DIM, generator=g)
    return types.SimpleNamespace(forward=lambda tokens, positions: table[tokens], output=lambda h: h @ weight.t(), loss_chunks=3, table=table, weight=weight)


@pytest.mark.parametrize("shape", [(2, 5), (1, 1), (3, 4)])
@pytest.mark.parametrize("several", [(), (1,), (4,)])
def test_targets_go_with_their_tokens(decoder, shape, several):
    g = torch.Generator().manual_seed(1)
    tokens, targets = torch.randint(0, VOCAB, shape, generator=g), torch.randint(0, VOCAB, (*shape, *several), generator=g)
    r = harness.Decoder.token_logprobs(decoder, tokens, targets, temperature=0.5, entropy=True, top=2)
    log_p = torch.log_softmax(decoder.table.double()[tokens] @ decoder.weight.double().t() / 0.5, -1)
    assert r.logprobs.shape == targets.shape and r.entropy.shape == shape and r.top_tokens.shape == (*shape, 2)
    for at in torch.cartesian_prod(*(torch.arange(n) for n in targets.shape)).reshape(-1, targets.dim()).tolist():
        assert abs(float(r.logprobs[tuple(at)]) - float(log_p[at[0], at[1], targets[tuple(at)]])) < 1e-4
    assert torch.equal(r.top_tokens, log_p.topk(2).indices)


@pytest.mark.parametrize("targets", [(2, 10), (5, 2), (4, 5), (10,), (2, 5, 1, 1), (2, 4), ()])
def test_targets_of_another_shape_are_refused(decoder, targets):
    """Twice as many would otherwise be two for each token, and others' at that."""
    with pytest.raises(ValueError, match="do not fit"):
        harness.Decoder.token_logprobs(decoder, torch.zeros(2, 5, dtype=torch.long), torch.zeros(targets, dtype=torch.long))
