"""What the serving classes do on the host, on the CPU: the device's calls are stand-ins that index as the device would,
so an index out of range raises here."""

from types import SimpleNamespace

import pytest
import torch

from pollux_amd import model as pm
from pollux_amd.model import GraphDecoder, PackedPolluxModel, PolluxConfig
from pollux_amd.paged import PagedKVCache
from pollux_amd.sampling import Sampling

CFG = PolluxConfig(vocab_size=240, tokenizer_vocab_size=230, seq_len=12, n_layers=1, n_heads=2, n_embd=48, d_head=24)


class _Step(GraphDecoder):
    """The decoder with its graphs run as plain steps."""

    captured = 0

    def _capture_prefill(self, T):
        ids = torch.zeros(self.ids.shape[0], T, dtype=torch.long)
        last = torch.zeros((), dtype=torch.long)
        return SimpleNamespace(replay=lambda: None), ids, last, torch.zeros(ids.shape[0], 1, CFG.vocab_size)

    def _capture(self):
        self.captured += 1
        saved = self.length
        self.pos.fill_(saved)
        self.logits = self._step()
        self.pos.fill_(saved)
        self.graph = SimpleNamespace(replay=self._step)


def _stand_ins(monkeypatch):
    model = PackedPolluxModel(CFG)
    model.blocks = torch.nn.ModuleList()
    model.embed = lambda idx, pos0: torch.zeros(*idx.shape, CFG.n_embd)
    model.logits = lambda x: torch.zeros(*x.shape[:2], CFG.vocab_size)
    monkeypatch.setattr(pm, "argmax_rows", lambda x, out: out.copy_(x.argmax(-1)))
    monkeypatch.setattr(pm, "sample_rows", lambda x, u, out, **rules: out.copy_((u * 100).long()))
    return model


@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("sampling", [True, False])
@pytest.mark.parametrize("max_len", [12, 7])
def test_a_prompt_that_fills_the_cache(monkeypatch, sampling, max_len, batch):
    model = _stand_ins(monkeypatch)
    monkeypatch.setattr(pm.PackedInt8Linear, "gemv_runs", lambda self, x: False)  # greedy: the argmax by its own call
    dec = _Step(model, batch=batch, max_len=max_len, greedy=not sampling, sampling=Sampling() if sampling else None)
    first = torch.zeros(batch, dtype=torch.long)

    def decode(n):
        return dec.decode_sampled(first, torch.full((batch, n), 0.5)) if sampling else dec.decode_greedy(first, n)

    with pytest.raises(RuntimeError, match="before prefill"):
        decode(1)
    with pytest.raises(RuntimeError, match="before prefill"):
        dec.decode(first)
    dec.prefill(torch.ones(batch, max_len, dtype=torch.long))  # no position is left for a step
    assert dec.captured == 0 and decode(0).shape == (batch, 0)
    with pytest.raises(ValueError, match="positions"):
        dec.decode(first)
    with pytest.raises(ValueError, match="positions"):
        decode(1)
    dec.prefill(torch.ones(batch, max_len - 2, dtype=torch.long))
    assert dec.captured == 1
    assert decode(2).tolist() == [[50, 50] if sampling else [0, 0]] * batch
    with pytest.raises(ValueError, match="positions"):
        decode(1)


def test_ids_that_name_no_token_give_nan_rows_of_materialized_weights():
    # as the packed embedding's kernel does: a row without a distribution draws the id -1, which a replay then embeds
    model = PackedPolluxModel(CFG)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        model.pos_emb.weight.copy_(torch.randn(CFG.seq_len, CFG.n_embd, generator=g))
    emb = model.tok_emb
    emb.weight = torch.nn.Parameter(torch.randn(CFG.vocab_size, CFG.n_embd, generator=g).half(), requires_grad=False)
    emb._materialized = True
    x = model.embed(torch.tensor([[3, 4], [-1, 239], [0, 240]]), torch.tensor(5)).detach()
    assert x.isnan().any(-1).tolist() == x.isnan().all(-1).tolist() == [[False, False], [True, False], [False, True]]
    for at, (t, p) in {(0, 0): (3, 5), (0, 1): (4, 6), (1, 1): (239, 6), (2, 0): (0, 5)}.items():
        assert torch.equal(x[at], emb.weight[t].float() + model.pos_emb.weight[p])


def test_settings_of_another_number_of_sequences():
    # (each step selects the settings of the sequences that draw, by index, on the device)
    model = PackedPolluxModel(CFG)
    for n in (1, 2, 4):
        with pytest.raises(ValueError, match="top_k must have 3 values"):
            pm.generate_many(model, [[1], [2, 3], [4]], sampling=Sampling(temperature=torch.ones(3), top_k=torch.ones(n).long()))
    with pytest.raises(ValueError, match="temperature must have 3 values"):
        pm.generate_many(model, [[1], [2, 3], [4]], sampling=Sampling(temperature=torch.ones(3, device="meta")))


def test_sequences_that_there_are_not():
    cache = PagedKVCache([SimpleNamespace(k=torch.zeros(4, 2, 8, 24), page_size=8, heads=2)])
    a, b = cache.add(), cache.add()
    cache.drop(b)
    for seq in (b, 99, -1):
        for call in (lambda: PackedPolluxModel(CFG).extend([[1], [2]], cache, [a, seq]), lambda: cache.length(seq),
                     lambda: cache.drop(seq), lambda: cache.extend([a, seq], [1, 1])):
            with pytest.raises(ValueError, match="no such sequence"):
                call()
    assert cache.free_pages == 4 and cache.length(a) == 0
