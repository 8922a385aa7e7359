"""The paged cache, its attention and the sampler as the model uses them: extend, generate_many, sampled generation.

Bars: logits over fp32 pages against the uncached forward, relative L2 <= 1e-5 (as the contiguous cache's); tokens of
prompts served together equal to those of each alone (fp32 pages).  INT8 pages move a key or value by up to 1/254 of its
row's largest: their logits are only held to 10%, a sanity bound, and fp16's (2^-11) to 1%.
"""

import pytest
import torch

from pollux_amd import pack, plx
from pollux_amd.model import GraphDecoder, PackedPolluxModel, generate, generate_many
from pollux_amd.paged import PagedKVCache
from pollux_amd.sampling import Sampling, sample_rows
from test_gpu_model import CFG, _dense_state

pytestmark = pytest.mark.gpu

BIG = {**CFG, "n_heads": 3, "n_embd": 72, "vocab_size": 240, "tokenizer_vocab_size": 230, "seq_len": 96}


@pytest.fixture(scope="module")
def model(dev, tmp_path_factory):
    state, _ = pack.pack_state_dict(_dense_state(BIG, 9), dev)
    path = tmp_path_factory.mktemp("plx") / "serving.plx"
    plx.write_plx(path, pack.pack_config(BIG), state)
    return PackedPolluxModel.from_packed_checkpoint(path, dev)


def _prompts(lengths, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, BIG["tokenizer_vocab_size"], (n,), generator=g).tolist() for n in lengths]


@pytest.mark.parametrize("kv_dtype,bar", [(torch.float32, 1e-5), (torch.float16, 1e-2), (torch.int8, 0.1)])
def test_extend_against_the_full_forward(model, dev, kv_dtype, bar):
    cache = PagedKVCache.allocate(model.cfg, 40, dev, page_size=8, kv_dtype=kv_dtype)
    prompts = _prompts([90, 3, 41, 70])
    seqs = [cache.add() for _ in prompts]
    done = [0] * 4
    # chunks of several sizes, single tokens, steps without some of the sequences
    for step in ([50, 2, 1, 0], [1, 1, 0, 33], [30, 0, 39, 1], [1, 0, 1, 1], [8, 0, 0, 35]):
        live = [i for i in range(4) if step[i]]
        tokens = [prompts[i][done[i]:done[i] + step[i]] for i in live]
        logits = model.extend(tokens, cache, [seqs[i] for i in live])
        for k, i in enumerate(live):
            done[i] += step[i]
            assert cache.length(seqs[i]) == done[i]
            with torch.inference_mode():
                ref = model(torch.tensor([prompts[i][:done[i]]], device=dev), last_only=True)[0, 0]
            rel = ((logits[k] - ref).norm() / ref.norm()).item()
            print(f"[serving] {kv_dtype} sequence {i} at {done[i]}: rel {rel:.2e}", flush=True)
            assert rel <= bar
    free = cache.free_pages
    cache.drop(seqs[0])
    assert cache.free_pages == free + 12  # 90 positions in pages of 8


def test_extend_with_materialized_weights(model, dev, tmp_path):
    state, _ = pack.pack_state_dict(_dense_state(BIG, 9), dev)
    plx.write_plx(tmp_path / "dense.plx", pack.pack_config(BIG), state)
    dense = PackedPolluxModel.from_packed_checkpoint(tmp_path / "dense.plx", dev, materialize=True)
    cache = PagedKVCache.allocate(dense.cfg, 40, dev, page_size=8, kv_dtype=torch.float32)
    prompts = _prompts([30, 1, 96])
    logits = dense.extend(prompts, cache, [cache.add() for _ in prompts])
    for got, p in zip(logits, prompts):
        with torch.inference_mode():
            ref = dense(torch.tensor([p], device=dev), last_only=True)[0, 0]
        assert ((got - ref).norm() / ref.norm()).item() <= 1e-5


def test_generate_many_equals_each_alone(model, dev):
    prompts = _prompts([5, 33, 1, 64])
    for sampling in (None, Sampling(temperature=0.9, top_k=20, top_p=0.9, min_p=0.01, repetition_penalty=1.1)):
        u = torch.rand(4, 12, generator=torch.Generator(device=dev).manual_seed(4), device=dev)
        got = generate_many(model, prompts, max_new_tokens=12, sampling=sampling, u=u, eos_id=229, chunk=16,
                            page_size=16, kv_dtype=torch.float32)
        for i, p in enumerate(prompts):
            greedy = Sampling(temperature=0.0)
            alone = generate(model, p, max_new_tokens=12, sampling=sampling or greedy, u=u[i].contiguous(), eos_id=229)
            assert got[i] == alone, i
        print(f"[serving] {[g[len(p):] for g, p in zip(got, prompts)]}", flush=True)
    # INT8 pages, settings of each prompt's own
    own = Sampling(temperature=torch.tensor([0.5, 1.0, 0.0, 2.0], device=dev), top_k=torch.tensor([3, 0, 0, 50], device=dev))
    got = generate_many(model, prompts, max_new_tokens=5, sampling=own, eos_id=-1)
    assert [len(g) - len(p) for g, p in zip(got, prompts)] == [5] * 4
    assert all(0 <= t < 230 for g in got for t in g)


def test_generate_many_at_the_end_of_the_context_and_of_the_pages(model, dev):
    prompts = _prompts([96, 90, 2])
    got = generate_many(model, prompts, max_new_tokens=9, eos_id=-1)
    assert [len(g) for g in got] == [97, 97, 11]  # the last token of a full context is drawn, not fed back
    cache = PagedKVCache.allocate(model.cfg, 13, dev, page_size=8)
    with pytest.raises(ValueError, match="pages needed"):
        generate_many(model, prompts, max_new_tokens=9, cache=cache)
    assert cache.free_pages == 13
    assert generate_many(model, prompts[2:], max_new_tokens=3, cache=cache, eos_id=-1)[0][:2] == prompts[2]
    assert cache.free_pages == 13
    assert generate_many(model, [], max_new_tokens=3) == [] and generate_many(model, prompts, max_new_tokens=0) == prompts


def test_sampled_generation_with_and_without_graph_and_cache(model, dev):
    prompt = _prompts([7])[0]
    u = torch.rand(30, generator=torch.Generator(device=dev).manual_seed(8), device=dev)
    rules = Sampling(temperature=0.8, top_k=30, top_p=0.95, repetition_penalty=1.2)
    runs = [generate(model, prompt, max_new_tokens=30, sampling=rules, u=u, eos_id=-1, use_cache=c, use_graph=g)
            for c, g in ((True, False), (True, True), (False, False))]
    assert runs[0] == runs[1] == runs[2]


def test_decode_sampled_follows_the_eager_steps(model, dev):
    prompts = torch.tensor(_prompts([9, 9]), device=dev)
    u = torch.rand(2, 20, generator=torch.Generator(device=dev).manual_seed(6), device=dev)
    rules = Sampling(temperature=0.9, top_p=0.9, repetition_penalty=1.3)
    dec = GraphDecoder(model, batch=2, sampling=rules)
    first = dec.prefill(prompts).argmax(-1)
    got = dec.decode_sampled(first, u[:, :12])
    got = torch.cat([got, dec.decode_sampled(got[:, -1], u[:, 12:])], 1)
    with torch.inference_mode():
        cache = model.new_cache(2)
        model.prefill(prompts, cache)
        seq = torch.cat([prompts, first.view(2, 1)], 1)
        for i in range(20):
            logits = model.decode(seq[:, -1], cache)
            ids = sample_rows(logits, u[:, i].contiguous(), temperature=0.9, top_p=0.9, repetition_penalty=1.3, seen=seq,
                              vocab=230)
            seq = torch.cat([seq, ids.view(2, 1)], 1)
    assert torch.equal(got, seq[:, 10:])
    # a second prompt on the same decoder forgets the first
    again = dec.prefill(prompts).argmax(-1)
    assert torch.equal(dec.decode_sampled(again, u[:, :12]), got[:, :12])


def test_refusals(model, dev):
    cache = PagedKVCache.allocate(model.cfg, 4, dev, page_size=16)
    a, b = cache.add(), cache.add()
    with pytest.raises(ValueError, match="pages needed"):
        cache.extend([a, b], [40, 30])
    assert cache.free_pages == 4 and cache.length(a) == 0
    for seqs, counts in (([a, a], [1, 1]), ([a], [0]), ([a, b], [1]), ([99], [1])):
        with pytest.raises(ValueError):
            cache.extend(seqs, counts)
    with pytest.raises(ValueError, match="token ids"):
        model.extend([[240]], cache, [a])
    with pytest.raises(ValueError, match="seq_len"):
        model.extend([[1] * 97], cache, [a])
    with pytest.raises(ValueError, match="not one of this model"):
        model.extend([[1]], PagedKVCache(cache.layers[:1]), [0])
    with pytest.raises(ValueError, match="not both"):
        GraphDecoder(model, greedy=True, sampling=Sampling())
    with pytest.raises(ValueError, match="not both"):
        generate(model, [1], sampling=Sampling(), sample=lambda x, i: 0)
    with pytest.raises(ValueError, match="u must be"):
        generate(model, [1], sampling=Sampling(), u=torch.zeros(3, device=dev))
    with pytest.raises(RuntimeError, match="sampling"):
        GraphDecoder(model).decode_sampled(torch.zeros(1, dtype=torch.long, device=dev), torch.zeros(1, 2, device=dev))
    for prompts in ([[]], [[1] * 97], [[240]]):
        with pytest.raises(ValueError):
            generate_many(model, prompts)
    assert cache.free_pages == 4


@pytest.mark.parametrize("sampling", [True, False])
@pytest.mark.parametrize("batch,max_len", [(1, 63), (2, 96)])
def test_a_decoder_whose_first_prompt_fills_the_cache(model, dev, sampling, batch, max_len, monkeypatch):
    monkeypatch.setattr(model.head, "gemv_max_tokens", 0 if not sampling else model.head.gemv_max_tokens)  # unfused greedy
    rules = Sampling(temperature=0.9, top_p=0.9)
    make = lambda: GraphDecoder(model, batch=batch, max_len=max_len, greedy=not sampling,  # noqa: E731
                                sampling=rules if sampling else None)
    u = torch.rand(batch, 5, generator=torch.Generator(device=dev).manual_seed(2), device=dev)

    def decode(dec, first, n):
        return dec.decode_sampled(first, u[:, :n]) if sampling else dec.decode_greedy(first, n)

    full = torch.tensor(_prompts([max_len] * batch), device=dev)
    dec, fresh = make(), make()
    logits = dec.prefill(full)
    with torch.inference_mode():
        want = model.prefill(full, model.new_cache(batch, max_len), last_only=True)[:, -1]
    assert ((logits - want).norm() / want.norm()).item() <= 1e-5
    assert decode(dec, logits.argmax(-1), 0).shape == (batch, 0)
    with pytest.raises(ValueError, match="positions"):
        decode(dec, logits.argmax(-1), 1)
    with pytest.raises(ValueError, match="positions"):
        dec.decode(logits.argmax(-1))
    got, ref = (decode(d, d.prefill(full[:, :-5]).argmax(-1), 5) for d in (dec, fresh))
    assert torch.equal(got, ref)
    assert torch.equal(decode(dec, dec.prefill(full[:, :-5]).argmax(-1), 5), got)


@pytest.mark.parametrize("batch", [3, 7, 40])
@pytest.mark.parametrize("materialize", [False, True])
def test_a_sequence_without_a_distribution_stays_without_one(model, dev, tmp_path, materialize, batch):
    if materialize:
        state, _ = pack.pack_state_dict(_dense_state(BIG, 9), dev)
        plx.write_plx(tmp_path / "dense.plx", pack.pack_config(BIG), state)
        model = PackedPolluxModel.from_packed_checkpoint(tmp_path / "dense.plx", dev, materialize=True)
    prompts = torch.tensor(_prompts([9] * batch), device=dev)
    u = torch.rand(batch, 12, generator=torch.Generator(device=dev).manual_seed(6), device=dev)
    others = [i for i in range(batch) if i != 1]
    got = []
    for middle in (0.7, float("nan")):  # the second sequence's temperature
        rules = Sampling(temperature=torch.tensor([0.9, middle] + [1.1] * (batch - 2), device=dev), top_p=0.95, repetition_penalty=1.2)
        dec = GraphDecoder(model, batch=batch, sampling=rules)
        ids = dec.decode_sampled(dec.prefill(prompts).argmax(-1), u[:, :7])
        got.append(torch.cat([ids, dec.decode_sampled(ids[:, -1], u[:, 7:])], 1))  # (its last ids fed back by hand)
    assert (got[0] >= 0).all() and (got[1][1] == -1).all()
    assert torch.equal(got[0][others], got[1][others])
    # a prefill starts afresh; then an id that is none, by the caller
    rules.temperature[1] = 0.7
    first = dec.prefill(prompts).argmax(-1)
    assert torch.equal(dec.decode_sampled(first, u[:, :7]), got[0][:, :7])
    first = dec.prefill(prompts).argmax(-1)
    first[1] = -1
    ids = dec.decode_sampled(first, u[:, :7])
    assert (ids[1] == -1).all() and torch.equal(ids[others], got[0][others, :7])
