"""LSTM language model (WikiText-2 shape).

Capability analog of the reference's RNN example
(reference: examples/wikitext_models.py; its trainer calls a stale K-FAC
API, examples/pytorch_wikitext_rnn.py:196-202 -- this one works against
the current API: the decoder Linear carries K-FAC factors, LSTM weights
stay first-order)."""

from __future__ import annotations

import torch
import torch.nn as nn

from kfac_pytorch_amd.ops.vocab_loss import projection_loss

__all__ = ["LSTMLanguageModel"]


class LSTMLanguageModel(nn.Module):
    def __init__(self, vocab_size: int = 33278, emb: int = 256,
                 hidden: int = 256, layers: int = 2, dropout: float = 0.5,
                 tie_weights: bool = True):
        super().__init__()
        self.drop = nn.Dropout(dropout)
        self.embed = nn.Embedding(vocab_size, emb)
        self.lstm = nn.LSTM(emb, hidden, layers, dropout=dropout,
                            batch_first=True)
        self.decoder = nn.Linear(hidden, vocab_size)
        if tie_weights:
            assert emb == hidden
            self.decoder.weight = self.embed.weight
        self.vocab_size = vocab_size

    def forward(self, x, hidden=None, targets=None, ignore_index=-100):
        """Logits and the LSTM's state; with ``targets`` (token numbers, the
        shape of ``x``) the mean cross entropy instead of the logits, which
        are then never in memory (``ops.linear_cross_entropy``).  Targets of
        ``ignore_index`` are left out."""
        emb = self.drop(self.embed(x))
        out, hidden = self.lstm(emb, hidden)
        out = self.drop(out)
        if targets is not None:
            return projection_loss(self.decoder, out, targets,
                                   ignore_index=ignore_index), hidden
        return self.decoder(out), hidden
