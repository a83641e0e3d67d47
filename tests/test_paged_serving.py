"""Paged cache bookkeeping, paged serving, packed forwards and scoring (CPU), and
the same runs on the kernels."""

import json
import math

import pytest
import torch

from luminaai_amd import ops
from luminaai_amd.inference import (ContinuousBatchingEngine,
                                    GenerationConfig, GenerationEngine,
                                    PagedBatchingEngine, PagedKVCache)


def _cfg(n=6, **kw):
    return GenerationConfig(max_new_tokens=n, temperature=0.0,
                            stop_token_ids=[-1], **kw)


def _engine(model, tokenizer, **kw):
    kw = {"max_batch": 4, "max_len": 64, "page_size": 16, **kw}
    return PagedBatchingEngine(model, tokenizer, **kw)


# ------------------------------------------------------------ bookkeeping
def _cache(pages=8, **kw):
    return PagedKVCache(2, 1, 8, pages, 16, max_seqs=4, max_len=80,
                        dtype=torch.float32, **kw)


def _check(c):
    """Reference counts are what the tables say, and the free pages the rest."""
    used = [p for t in c.tables for p in t]
    assert c._refs == [used.count(p) for p in range(c.pages)]
    assert sorted(c._free) == [p for p in range(c.pages) if not c._refs[p]]
    for slot, t in enumerate(c.tables):
        assert c._table[slot, :len(t)].tolist() == t
        assert len(t) == c.pages_for(c.lens[slot])


def _write(c, slot, value):
    """One token of `value` into every layer."""
    layers = c.decode([slot])
    for i, layer in enumerate(layers):
        kv = torch.full((1, 1, 8), value + i)
        layer.append(kv, -kv)


def _read(c, slot):
    pages = torch.tensor(c.tables[slot])
    return [c.k[i][pages].transpose(1, 2).reshape(-1, 8)[:c.lens[slot], 0]
            .tolist() for i in range(2)]


def test_cache_grow_fork_free_compact_resize():
    c = _cache()
    c.prefill([1], [20])
    _check(c)
    for t in range(15):
        _write(c, 0, 100.0 + t)
    _write(c, 1, 7.0)
    _check(c)
    c.fork(0, 2)
    c.fork(0, 3)
    _check(c)
    assert c.tables[2] == c.tables[0] and c.free_pages == 8 - 3
    # the first two writers copy the shared page, the last one keeps it
    assert c.pages_needed([0, 2, 3], [1, 1, 1]) == 2
    for slot, v in ((0, 1.0), (2, 2.0), (3, 3.0)):
        _write(c, slot, v)
        _check(c)
    assert len({c.tables[s][0] for s in (0, 2, 3)}) == 3
    base = [100.0 + t for t in range(15)]
    for slot, v in ((0, 1.0), (2, 2.0), (3, 3.0)):
        assert _read(c, slot) == [base + [v], [x + 1 for x in base] + [v + 1]]
    one = _read(c, 1)
    c.free(0)
    c.free(2)
    _check(c)
    assert c.compact() == 0         # the live pages are the first already
    _write(c, 0, 5.0)
    assert _read(c, 1) == one
    c.free(1)
    assert c.compact() == 2
    _check(c)
    assert sorted(p for t in c.tables for p in t) == [0, 1]
    assert _read(c, 3)[0] == base + [3.0] and _read(c, 0) == [[5.0], [6.0]]
    c.resize(2)
    _check(c)
    assert _read(c, 3)[0] == base + [3.0] and c.free_pages == 0
    with pytest.raises(ValueError, match="in use"):
        c.resize(1)
    c.resize(9)
    _check(c)
    _write(c, 3, 4.0)
    assert _read(c, 3)[0] == base + [3.0, 4.0]
    assert _read(c, 0) == [[5.0], [6.0]]


@pytest.mark.parametrize("held", [0, 5, 16, 20])
def test_room_made_ahead_is_not_shared(held):
    """extend() takes pages before they are written; a fork shares what is
    written and nothing else."""
    c = _cache()
    for t in range(held):
        _write(c, 0, 100.0 + t)
    c.extend([0], [40])
    c.fork(0, 1)
    used = [p for t in c.tables for p in t]
    assert c._refs == [used.count(p) for p in range(c.pages)]
    assert len(c.tables[1]) == c.pages_for(held)
    for t in range(20):
        _write(c, 0, 200.0 + t)
        _write(c, 1, 300.0 + t)
    base = [100.0 + t for t in range(held)]
    assert _read(c, 0)[0] == base + [200.0 + t for t in range(20)]
    assert _read(c, 1)[0] == base + [300.0 + t for t in range(20)]
    c.free(0)
    c.free(1)
    assert c.free_pages == c.pages


def test_cache_refusals_change_nothing():
    c = _cache(pages=2)
    c.prefill([0], [17])
    for call, err in [(lambda: c.prefill([1], [1]), MemoryError),
                      (lambda: c.extend([0], [64]), ValueError),
                      (lambda: c.decode([0, 0]), ValueError),
                      (lambda: c.prefill([0], [1]), ValueError),
                      (lambda: c.fork(1, 0), ValueError)]:
        with pytest.raises(err):
            call()
        _check(c)
        assert c.lens == [17, 0, 0, 0]
    with pytest.raises(ValueError, match="power of two"):
        PagedKVCache(1, 1, 8, 4, 24)


# ------------------------------------------------------------ packed forward
def test_packed_forward_equals_each_alone(small_model):
    m = small_model.eval()
    g = torch.Generator().manual_seed(0)
    seqs = [torch.randint(1, 500, (n,), generator=g) for n in (5, 1, 17, 30)]
    cu = torch.tensor([0, 5, 6, 23, 53], dtype=torch.int32)
    with torch.no_grad():
        out, _, _ = m(torch.cat(seqs)[None], cu_seqlens=cu)
        for i, s in enumerate(seqs):
            alone, _, _ = m(s[None])
            assert torch.allclose(out[0, cu[i]:cu[i + 1]], alone[0],
                                  atol=1e-5)


@pytest.mark.parametrize("checkpointing", [False, True])
def test_packed_training_equals_padded(small_model, tiny_config,
                                       checkpointing):
    """Loss and gradients of a packed batch are those of the padded one."""
    from luminaai_amd.data import pack_collate
    from luminaai_amd.ops import fused_cross_entropy
    m = small_model.train()
    m.gradient_checkpointing = checkpointing
    g = torch.Generator().manual_seed(1)
    samples = []
    for n in (3, 11, 20):
        ids = torch.zeros(21, dtype=torch.long)
        ids[:n + 1] = torch.randint(1, 500, (n + 1,), generator=g)
        labels = ids[1:].clone()
        labels[n:] = -100
        samples.append({"input_ids": ids[:-1], "labels": labels,
                        "loss_weights": torch.rand(20, generator=g)})
    grads = []
    for batch in (torch.utils.data.default_collate(samples),
                  pack_collate(samples)):
        kw = {k: v for k, v in batch.items() if k == "cu_seqlens"}
        logits, _, _ = m(batch["input_ids"], **kw)
        loss, _, n = fused_cross_entropy(logits, batch["labels"],
                                         batch["loss_weights"])
        grads.append((loss, torch.autograd.grad(loss, list(m.parameters())),
                      int(n)))
    assert grads[0][2] == grads[1][2] == 34
    assert torch.allclose(grads[0][0], grads[1][0], atol=1e-6)
    for a, b in zip(grads[0][1], grads[1][1]):
        assert torch.allclose(a, b, atol=1e-6)


def test_trainer_takes_packed_batches(tiny_config, sample_conversations,
                                      tokenizer):
    from luminaai_amd.data import ConversationDataset, create_dataloader
    from luminaai_amd.models import (DeepSeekTransformer,
                                     config_to_deepseek_config)
    from luminaai_amd.training import Trainer
    tiny_config.pack_sequences = True
    torch.manual_seed(0)
    m = DeepSeekTransformer(config_to_deepseek_config(tiny_config))
    ds = ConversationDataset(sample_conversations, tokenizer, 64)
    loader = create_dataloader(ds, tiny_config, shuffle=False)
    batch = next(iter(loader))
    assert batch["input_ids"].shape[0] == 1
    assert batch["cu_seqlens"].tolist()[-1] == batch["input_ids"].shape[1]
    t = Trainer(m, tokenizer, tiny_config)
    t._setup_scheduler(4)
    out = t.train_step(batch)
    t.optimizer_step()
    assert math.isfinite(float(out["ce_loss"]))
    res = t.evaluate(loader)
    assert math.isfinite(res["loss"])


def _moe(cfg):
    from luminaai_amd.models import (DeepSeekTransformer,
                                     config_to_deepseek_config)
    torch.manual_seed(0)
    return DeepSeekTransformer(config_to_deepseek_config(cfg))


def test_packed_moe(tiny_moe_config):
    """Experts see the tokens of all sequences, which attend to themselves."""
    m = _moe(tiny_moe_config).train()
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(1, 500, (1, 30), generator=g)
    cu = torch.tensor([0, 12, 30], dtype=torch.int32)
    logits, aux, _ = m(ids, cu_seqlens=cu)
    grads = torch.autograd.grad(logits.float().square().mean() + aux,
                                list(m.parameters()), allow_unused=True)
    assert all(x is None or bool(x.isfinite().all()) for x in grads)


def _dropping_moe(cfg):
    """Experts that many tokens want: a forward drops a good part of them."""
    cfg.num_layers, cfg.num_experts, cfg.seq_length = 3, 8, 64
    m = _moe(cfg).eval()
    g = torch.Generator().manual_seed(7)
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() > 1:
                p.copy_(0.2 * torch.randn(p.shape, generator=g))
    return m


def _sequences(*lens):
    g = torch.Generator().manual_seed(5)
    return [torch.randint(1, 500, (n,), generator=g).tolist() for n in lens]


def test_moe_forward_of_each_packed_sequence_is_its_own(tiny_moe_config):
    m = _dropping_moe(tiny_moe_config)
    seqs = [torch.tensor(s) for s in _sequences(12, 1, 60, 33)]
    cu = torch.tensor([0, 12, 13, 13, 73, 106], dtype=torch.int32)
    pad = torch.ones(4, dtype=torch.long)        # behind the last sequence
    with torch.no_grad():
        out = m(torch.cat([*seqs, pad])[None], cu_seqlens=cu)[0][0]
        at = 0
        for s in seqs:
            alone = m(s[None])[0][0]
            assert torch.allclose(out[at:at + len(s)], alone, atol=1e-4)
            at += len(s)


def test_moe_scores_do_not_depend_on_the_batch(tiny_moe_config, tokenizer):
    solo = GenerationEngine(_dropping_moe(tiny_moe_config), tokenizer)
    seqs = _sequences(12, 33, 60, 25)
    for s, r in zip(seqs, solo.score(seqs)):
        alone = solo.score([s])[0]
        for k in ("logprobs", "entropy"):
            assert torch.allclose(torch.tensor(r[k]), torch.tensor(alone[k]),
                                  atol=1e-4)


def test_paged_moe_answers_do_not_depend_on_the_batch(tiny_moe_config,
                                                      tokenizer):
    m = _dropping_moe(tiny_moe_config)
    prompts = _sequences(12, 33, 40, 25)
    solo = GenerationEngine(m, tokenizer)
    refs = [solo.generate(p, _cfg(8)) for p in prompts]
    eng = _engine(m, tokenizer)
    assert eng.run_to_completion(prompts, _cfg(8)) == refs
    assert eng.run_to_completion(prompts, _cfg(8),
                                 admit_schedule=[0, 2, 2, 5]) == refs


def test_paged_engine_with_quantized_moe(tiny_moe_config, tokenizer):
    from luminaai_amd.ops.quant import quantize_model
    m = _moe(tiny_moe_config).eval()
    quantize_model(m, mode="int8", min_dim=32)
    eng = _engine(m, tokenizer, max_batch=2)
    outs = eng.run_to_completion([tokenizer.encode("quantized"),
                                  tokenizer.encode("serving")], _cfg(4))
    assert all(len(o) == 4 and all(isinstance(t, int) for t in o)
               for o in outs)


@pytest.mark.parametrize("cu", [[0, 3, 8], [5, 6, 8], [0, 9, 2, 5], [0, 99],
                                [-40, 2, 8], [8, 8], [0]])
def test_positions_index_inside_the_row(cu):
    """Whatever the borders hold, positions stay below the row's length."""
    pos = ops.packed_positions(torch.tensor(cu, dtype=torch.int32), 8)
    assert pos.shape == (1, 8) and pos.dtype == torch.int32
    assert 0 <= int(pos.min()) and int(pos.max()) < 8
    if cu == [0, 3, 8]:
        assert pos[0].tolist() == [0, 1, 2, 0, 1, 2, 3, 4]


def test_packed_forward_refusals(small_model, tiny_config):
    from luminaai_amd.models import (DeepSeekTransformer,
                                     config_to_deepseek_config)
    ids = torch.ones(1, 6, dtype=torch.long)
    cu = torch.tensor([0, 2, 6], dtype=torch.int32)
    m = small_model.eval()
    with pytest.raises(ValueError, match="one row"):
        m(ids.expand(2, 6), cu_seqlens=cu)
    with pytest.raises(ValueError, match="no attention_mask"):
        m(ids, attention_mask=torch.ones(1, 6), cu_seqlens=cu)
    with pytest.raises(ValueError, match="no attention_mask"):
        m(ids, kv_caches=m.make_kv_caches(8), cu_seqlens=cu)
    c = PagedKVCache(2, 2, 16, 4, 16, dtype=torch.float32)
    layers, _ = c.prefill([0], [6])
    with pytest.raises(ValueError, match="packed prompts"):
        m(ids, kv_caches=layers)
    tiny_config.use_mod = True
    mod = DeepSeekTransformer(config_to_deepseek_config(tiny_config))
    with pytest.raises(ValueError, match="mixture-of-depths"):
        mod(ids, cu_seqlens=cu)
    tiny_config.use_mod = False
    tiny_config.dropout = 0.1
    drop = DeepSeekTransformer(config_to_deepseek_config(tiny_config)).train()
    with pytest.raises(ValueError, match="dropout"):
        drop(ids, cu_seqlens=cu)


# ------------------------------------------------------------ serving
def test_paged_matches_solo_staggered(small_model, tokenizer):
    solo = GenerationEngine(small_model.eval(), tokenizer)
    prompts = [tokenizer.encode(p) for p in
               ("the first and longest prompt here", "second one", "third",
                "a", "and one that comes when a slot is free again")]
    refs = [solo.generate(p, _cfg()) for p in prompts]
    eng = _engine(small_model, tokenizer, max_batch=3)
    outs = eng.run_to_completion(prompts, _cfg(),
                                 admit_schedule=[0, 2, 0, 9, 1])
    assert outs == refs
    assert eng.stats["admitted"] == eng.stats["finished"] == 5
    assert eng.cache.free_pages == eng.cache.pages
    _check(eng.cache)


def test_long_prompt_joins_at_once(small_model, tokenizer):
    """No admission waits for the others' length."""
    eng = _engine(small_model, tokenizer)
    a = eng.admit(tokenizer.encode("ab"), _cfg(8))
    eng.step()
    long = tokenizer.encode("a much longer prompt than two tokens")
    assert eng.can_admit(len(long))
    b = eng.admit(long, _cfg(3))
    while eng.n_active():
        eng.step()
    solo = GenerationEngine(small_model.eval(), tokenizer)
    assert eng.slots[b].result == solo.generate(long, _cfg(3))
    assert eng.slots[a].result == solo.generate(tokenizer.encode("ab"),
                                                _cfg(8))


def test_forks_continue_on_shared_pages(small_model, tokenizer):
    """Forks that decode greedily agree with solo; then one of them is led
    elsewhere and the others do not notice."""
    prompt = tokenizer.encode("a prompt that is forked in the middle of a page")
    solo = GenerationEngine(small_model.eval(), tokenizer)
    ref = solo.generate(prompt, _cfg(6))
    eng = _engine(small_model, tokenizer)
    a = eng.admit(prompt, _cfg(6))
    used = eng.cache.pages - eng.cache.free_pages
    b, c = eng.fork(a), eng.fork(a)
    assert eng.cache.pages - eng.cache.free_pages == used
    eng.last_logits[c] = 0
    eng.last_logits[c, ref[0] + 1] = 9.0
    while eng.n_active():
        eng.step()
    assert eng.slots[a].result == eng.slots[b].result == ref
    other = solo.generate(prompt + [ref[0] + 1], _cfg(5))
    assert eng.slots[c].result == [ref[0] + 1] + other
    _check(eng.cache)


def test_full_pool_ends_a_sequence(small_model, tokenizer):
    eng = _engine(small_model, tokenizer, pages=2)
    a = eng.admit([5] * 10, _cfg(60))
    b = eng.admit([6] * 12, _cfg(60))
    assert not eng.can_admit(1)
    while eng.n_active():
        eng.step()
    got = sorted(len(eng.slots[s].result) for s in (a, b))
    assert got[0] < got[1] and _check(eng.cache) is None
    with pytest.raises(RuntimeError, match="does not hold"):
        eng.run_to_completion([[5] * 40], _cfg(2))


def test_continuous_and_paged_agree(small_model, tokenizer):
    prompts = [tokenizer.encode(f"prompt number {i}") for i in range(4)]
    a = ContinuousBatchingEngine(small_model.eval(), tokenizer, max_batch=2,
                                 max_len=64)
    b = _engine(small_model, tokenizer, max_batch=2)
    assert a.run_to_completion(prompts, _cfg(4)) == \
        b.run_to_completion(prompts, _cfg(4))


def test_logprobs_of_answers_equal_scores(small_model, tokenizer):
    """What the engine reports while it decodes is what scoring the finished
    text says."""
    prompts = [tokenizer.encode("some prompt"), tokenizer.encode("x")]
    eng = _engine(small_model, tokenizer)
    slots = eng.admit_many(prompts, [_cfg(5, logprobs=3), _cfg(4)])
    while eng.n_active():
        eng.step()
    s = eng.slots[slots[0]]
    assert eng.slots[slots[1]].logprobs == []
    assert [e["token"] for e in s.logprobs] == s.result
    solo = GenerationEngine(small_model.eval(), tokenizer)
    full = prompts[0] + s.result
    score, empty, one = solo.score([full, [], [3]], top_k=3)
    assert empty["logprobs"] == [] and one["logprobs"] == []
    assert len(score["logprobs"]) == len(full) - 1
    for i, e in enumerate(s.logprobs):
        at = len(prompts[0]) - 1 + i
        assert abs(e["logprob"] - score["logprobs"][at]) < 1e-4
        assert [t for t, _ in e["top"]] == score["top_ids"][at]
        assert e["top"][0][0] == e["token"]         # greedy
    with pytest.raises(ValueError, match="logprobs"):
        eng.admit([1, 2], _cfg(2, logprobs=65))
    with pytest.raises(ValueError, match="outside the vocabulary"):
        eng.admit([1, 512])
    with pytest.raises(ValueError, match="outside the vocabulary"):
        solo.score([[1], [-1, 2]])


def test_scores_do_not_depend_on_the_batch(small_model, tokenizer):
    """More than one forward's worth of sequences, and each alone."""
    g = torch.Generator().manual_seed(0)
    seqs = [torch.randint(1, 500, (n,), generator=g).tolist()
            for n in (17, 2, 60)]
    solo = GenerationEngine(small_model.eval(), tokenizer)
    alone = [solo.score([s])[0]["logprobs"] for s in seqs]
    many = solo.score(seqs * 420)                   # 33180 tokens
    assert len(many) == 1260
    for i, r in enumerate(many):
        assert torch.allclose(torch.tensor(r["logprobs"]),
                              torch.tensor(alone[i % 3]), atol=1e-4)


def test_scores_of_empty_sequences(small_model, tokenizer):
    """Wherever they stand, and more of them than a packed row takes."""
    solo = GenerationEngine(small_model.eval(), tokenizer)
    want = solo.score([[1, 2]])[0]["logprobs"]
    assert solo.score([]) == []
    for seqs in ([[]], [[], [1, 2]], [[1, 2], []], [[], [], [1, 2], [5], []]):
        out = solo.score(seqs, top_k=2)
        assert [len(o["logprobs"]) for o in out] == \
            [max(0, len(s) - 1) for s in seqs]
        assert [len(o["top_ids"]) for o in out] == \
            [max(0, len(s) - 1) for s in seqs]
        for s, o in zip(seqs, out):
            if s == [1, 2]:
                assert abs(o["logprobs"][0] - want[0]) < 1e-5
    out = solo.score([[1, 2]] + [[]] * 65536 + [[1, 2]])
    assert len(out) == 65538
    assert abs(out[-1]["logprobs"][0] - want[0]) < 1e-5


def test_scores_one_by_one_for_wide_heads(tiny_config, tokenizer):
    from luminaai_amd.models import (DeepSeekTransformer,
                                     config_to_deepseek_config)
    tiny_config.hidden_size, tiny_config.num_heads = 400, 2
    tiny_config.num_kv_heads = 1                       # heads of 200
    torch.manual_seed(0)
    m = DeepSeekTransformer(config_to_deepseek_config(tiny_config)).eval()
    out = GenerationEngine(m, tokenizer).score([[], [1, 2, 3], [4, 5]])
    assert [len(o["logprobs"]) for o in out] == [0, 2, 1]
    with torch.no_grad():
        lp = m(torch.tensor([[1, 2, 3]]))[0][0].float().log_softmax(-1)
    assert abs(out[1]["logprobs"][1] - float(lp[1, 3])) < 1e-5


def test_alternatives_of_a_small_vocabulary(tiny_config, tokenizer):
    from luminaai_amd.models import (DeepSeekTransformer,
                                     config_to_deepseek_config)
    tiny_config.vocab_size = 40
    m = DeepSeekTransformer(config_to_deepseek_config(tiny_config)).eval()
    eng = _engine(m, tokenizer)
    eng._pad = 0
    b = eng.admit([1, 2, 3], _cfg(2, logprobs=64))
    while eng.n_active():
        eng.step()
    assert [len(e["top"]) for e in eng.slots[b].logprobs] == [40, 40]


def test_scores_one_by_one_for_mixture_of_depths(tiny_config, tokenizer):
    from luminaai_amd.models import (DeepSeekTransformer,
                                     config_to_deepseek_config)
    tiny_config.use_mod = True
    torch.manual_seed(0)
    m = DeepSeekTransformer(config_to_deepseek_config(tiny_config)).eval()
    out = GenerationEngine(m, tokenizer).score([[1, 2, 3], [4, 5]])
    assert [len(o["logprobs"]) for o in out] == [2, 1]
    with torch.no_grad():
        lp = m(torch.tensor([[1, 2, 3]]))[0][0].float().log_softmax(-1)
    assert abs(out[0]["logprobs"][1] - float(lp[1, 3])) < 1e-5


def test_server_paged(small_model, tokenizer):
    pytest.importorskip("fastapi")
    from fastapi.testclient import TestClient
    from luminaai_amd.inference.server import create_app
    client = TestClient(create_app(small_model.eval(), tokenizer,
                                   serving="paged", max_len=64, max_batch=4))
    body = {"prompt": "hello", "max_tokens": 4, "temperature": 0.0}
    one = client.post("/v1/completions", json=body).json()
    r = client.post("/v1/completions", json={**body, "n": 3, "logprobs": 2})
    got = r.json()
    assert r.status_code == 200 and len(got["choices"]) == 3
    for c in got["choices"]:
        assert c["text"] == one["choices"][0]["text"]
        assert len(c["logprobs"]["token_logprobs"]) == \
            one["usage"]["completion_tokens"]
    assert "logprobs" not in one["choices"][0]
    chat = client.post("/v1/chat/completions", json={
        "messages": [{"role": "user", "content": "hi"}], "max_tokens": 3,
        "temperature": 0.0, "logprobs": True, "top_logprobs": 1}).json()
    assert all(len(e["top_logprobs"]) == 1
               for e in chat["choices"][0]["logprobs"]["content"])
    for bad in ({"n": 9}, {"n": 0}, {"n": "x"}, {"logprobs": 65},
                {"logprobs": [1]}, {"n": 2, "stream": True}):
        assert client.post("/v1/completions",
                           json={**body, **bad}).status_code == 400
    lines = client.post("/v1/completions", json={**body, "stream": True}).text
    assert "text_completion.chunk" in lines
    # other modes answer once, as they always did
    plain = TestClient(create_app(small_model.eval(), tokenizer, max_len=64))
    got = plain.post("/v1/completions",
                     json={**body, "n": 2, "logprobs": 1}).json()
    assert [c["text"] for c in got["choices"]] == [one["choices"][0]["text"]]


def _worker(model, tokenizer, paged=True, **kw):
    from luminaai_amd.inference.server import _ContinuousWorker
    return _ContinuousWorker(model.eval(), tokenizer, max_len=64, paged=paged,
                             **{"max_batch": 3, **kw})


@pytest.mark.timeout(60)
@pytest.mark.parametrize("paged", [True, False])
def test_a_bad_request_leaves_the_server_as_it_was(small_model, tokenizer,
                                                   paged):
    """On a fresh server and on slots that were used before."""
    w = _worker(small_model, tokenizer, paged)
    want = GenerationEngine(small_model.eval(), tokenizer).generate([5, 6, 7],
                                                                    _cfg(4))
    for _ in range(4):                      # more than there are slots
        with pytest.raises(Exception, match="unhashable|whole numbers"):
            w.submit([1, 2, 3], GenerationConfig(stop_token_ids=[[1]]))
        assert w.eng.n_active() == 0
        assert w.submit([5, 6, 7], _cfg(4)) == want
    if paged:
        assert w.eng.cache.free_pages == w.eng.cache.pages


@pytest.mark.timeout(60)
def test_a_request_that_cannot_be_sampled_fails_alone(small_model, tokenizer):
    """temperature is not a number: the answer beside it goes on."""
    import threading
    w = _worker(small_model, tokenizer)
    want = GenerationEngine(small_model.eval(), tokenizer).generate([5, 6, 7],
                                                                    _cfg(30))
    got = []
    first = threading.Event()
    t = threading.Thread(target=lambda: got.append(
        w.submit([5, 6, 7], _cfg(30), lambda _: first.set())))
    t.start()
    assert first.wait(30)
    for n in (1, 2):
        with pytest.raises(RuntimeError):
            w.submit_n([1, 2], GenerationConfig(temperature=math.nan), n)
    t.join(30)
    assert got == [want]
    assert w.submit([5, 6, 7], _cfg(30)) == want
    assert w.eng.cache.free_pages == w.eng.cache.pages


def test_stop_tokens_of_any_integer_type(small_model, tokenizer):
    import numpy as np
    solo = GenerationEngine(small_model.eval(), tokenizer)
    stop = solo.generate([5, 6, 7], _cfg(6))[0]
    eng = _engine(small_model, tokenizer)
    for t in (stop, np.int64(stop), torch.tensor(stop)):
        cfg = GenerationConfig(max_new_tokens=6, temperature=0.0,
                               stop_token_ids=[t])
        # a list may be longer than the prompts are
        b, = eng.admit_many([[5, 6, 7]], [cfg, None], [None, None])
        while eng.n_active():
            eng.step()
        assert eng.slots[b].result == []


@pytest.mark.parametrize("bad", [2.5, "3", 65, -1])
def test_log_probabilities_of_one_row_do_not_end_the_others(
        small_model, tokenizer, bad):
    """One call computes those of all rows, so a bad number is refused before."""
    eng = _engine(small_model, tokenizer)
    a = eng.admit([1, 2, 3], _cfg(4, logprobs=1))
    with pytest.raises(ValueError, match="logprobs"):
        eng.admit([1, 2], _cfg(4, logprobs=bad))
    while eng.n_active():
        eng.step()
    assert eng.slots[a].error is None and len(eng.slots[a].logprobs) == 4


def test_engine_takes_nothing_for_a_request_it_refuses(small_model, tokenizer):
    eng = _engine(small_model, tokenizer)
    a = eng.admit([1, 2, 3], _cfg(4, logprobs=1))
    free, slots = eng.cache.free_pages, eng.free_slots()
    bad = GenerationConfig(stop_token_ids=["x"])
    for call in (lambda: eng.admit([1, 2], bad), lambda: eng.fork(a, bad),
                 lambda: eng.admit_many([[1], [2]], [None, bad]),
                 lambda: eng.admit_many([[1], [2]], [None]),
                 lambda: eng.admit_many([[1], [2]], None, [None])):
        with pytest.raises(ValueError):
            call()
        assert (eng.cache.free_pages, eng.free_slots()) == (free, slots)
        _check(eng.cache)
    # what fails while a row's log probabilities are taken ends that row
    b = eng.admit([4, 5], _cfg(4))
    eng.slots[a].cfg.logprobs = "x"
    while eng.n_active():
        eng.step()
    assert isinstance(eng.slots[a].error, TypeError)
    assert eng.slots[a].result == [] and eng.slots[b].error is None
    assert len(eng.slots[b].result) == 4
    with pytest.raises(RuntimeError):
        eng.run_to_completion([[1, 2]],
                              GenerationConfig(temperature=math.nan))


@pytest.mark.timeout(60)
@pytest.mark.parametrize("serving", ["paged", "continuous", "dynamic"])
def test_server_refuses_malformed_options(small_model, tokenizer, serving):
    pytest.importorskip("fastapi")
    from fastapi.testclient import TestClient
    from luminaai_amd.inference.server import create_app
    client = TestClient(create_app(small_model.eval(), tokenizer,
                                   serving=serving, max_len=64, max_batch=2),
                        raise_server_exceptions=False)
    ask = {"/v1/completions": {"prompt": "hello"},
           "/v1/chat/completions": {"messages": [{"role": "user",
                                                  "content": "hi"}]}}
    for path, body in ask.items():
        for bad in ('"stop_token_ids": [[1]]', '"stop_token_ids": ["a"]',
                    '"stop_token_ids": 3', '"stop_token_ids": null',
                    '"temperature": NaN', '"temperature": Infinity',
                    '"temperature": "warm"', '"max_tokens": null',
                    '"max_tokens": 1e999', '"top_p": NaN',
                    '"repetition_penalty": 0'):
            text = json.dumps({"max_tokens": 2, **body})[:-1] + f", {bad}}}"
            r = client.post(path, content=text,
                            headers={"content-type": "application/json"})
            assert r.status_code == 400, (path, bad, r.text)
        for good in ({"temperature": 1e-30}, {"stop_token_ids": [1]},
                     {"top_k": -1}):
            r = client.post(path, json={"max_tokens": 2, **body, **good})
            assert r.status_code == 200, (path, good, r.text)


class _Gate:
    """Lets the server's loop take one step at a time."""

    def __init__(self, worker):
        import threading
        self.worker = worker
        self.free = threading.Semaphore(0)
        self.at = threading.Semaphore(0)       # the loop waits before a step
        step = worker.eng.step

        def gated():
            self.at.release()
            assert self.free.acquire(timeout=30)
            return step()
        worker.eng.step = gated
        self.threads = []

    def ask(self, ids, cfg, n=1):
        """A request in a thread of its own; its result or exception."""
        import threading
        import time
        got = []

        def run():
            try:
                got.append(self.worker.submit_n(ids, cfg, n))
            except Exception as e:  # noqa: BLE001
                got.append(e)
        before = self.worker.q.qsize()
        busy = bool(self.threads)
        self.threads.append(threading.Thread(target=run, daemon=True))
        self.threads[-1].start()
        while busy and self.worker.q.qsize() == before:  # in order of asking
            time.sleep(0.001)
        return got

    def step(self, n=1):
        for _ in range(n):
            self.free.release()
            assert self.at.acquire(timeout=30)

    def run(self):
        """Until every request is answered."""
        for _ in range(1000):
            self.free.release()
        for t in self.threads:
            t.join(30)
            assert not t.is_alive()


def _got(answers):
    """What the thread of a request was answered."""
    import time
    end = time.monotonic() + 30
    while not answers and time.monotonic() < end:
        time.sleep(0.001)
    return answers[0]


@pytest.mark.timeout(60)
def test_server_refuses_what_never_fits_at_once(small_model, tokenizer):
    """While another request is served."""
    gate = _Gate(_worker(small_model, tokenizer))
    a = gate.ask([5, 6], _cfg(40))
    assert gate.at.acquire(timeout=30)
    long = gate.ask([5] * 64, _cfg(2))          # max_len is 64
    many = gate.ask([5, 6], _cfg(2), 4)         # of 3 slots
    gate.step(3)
    assert not a
    for r in (long, many):
        assert isinstance(_got(r), RuntimeError) and "context" in str(r[0])
    fits = gate.ask([5] * 63, _cfg(5))
    gate.run()
    # one more token finds room in the cache, and one is drawn behind it
    assert len(a[0][0][0]) == 40 and len(fits[0][0][0]) == 2


@pytest.mark.timeout(60)
def test_server_keeps_the_order_of_arrival(small_model, tokenizer):
    """A request for three answers waits for three slots, and single ones that
    come later do not take them as they are freed."""
    gate = _Gate(_worker(small_model, tokenizer))
    eng = gate.worker.eng
    a = gate.ask([5, 6], _cfg(3))
    assert gate.at.acquire(timeout=30)
    b = gate.ask([5, 7], _cfg(6))
    gate.step()
    three = gate.ask([5, 8], _cfg(4), 3)
    ones = [gate.ask([5, i], _cfg(4)) for i in range(9, 14)]
    gate.step(4)                                # a's slot is free again
    assert _got(a) and not b and eng.n_active() == 1
    gate.step(4)
    assert _got(b) and eng.n_active() == 3 and eng.stats["admitted"] == 5
    gate.run()
    assert [len(t) for t, _ in three[0]] == [4, 4, 4]
    assert all(len(o[0][0][0]) == 4 for o in ones)


@pytest.mark.timeout(60)
def test_server_prefills_together_what_comes_together(small_model, tokenizer):
    """One forward for the prompts that wait, forks besides; a bad one among
    them does not take the others along, and what never fits is refused though
    another waits before it."""
    gate = _Gate(_worker(small_model, tokenizer, max_batch=6))
    eng = gate.worker.eng
    sizes, admit = [], eng.admit_many
    eng.admit_many = lambda p, *a: sizes.append(len(p)) or admit(p, *a)
    solo = GenerationEngine(small_model.eval(), tokenizer)
    a = gate.ask([5, 6], _cfg(12))
    assert gate.at.acquire(timeout=30)
    prompts = [[7, 8, 9], [10], [11] * 20]
    got = [gate.ask(p, _cfg(4), n) for p, n in zip(prompts, (1, 2, 1))]
    gate.step()
    assert sizes == [1, 3] and eng.n_active() == 5
    gate.step(6)
    assert all(_got(g) for g in got) and not a
    late = [gate.ask([12], _cfg(4)), gate.ask([10 ** 6], _cfg(4)),
            gate.ask([13], _cfg(4), 6), gate.ask([3] * 70, _cfg(4))]
    gate.step()
    assert sizes == [1, 3, 2, 1, 1] and eng.n_active() == 2
    assert isinstance(_got(late[1]), ValueError)
    assert isinstance(_got(late[3]), RuntimeError)
    gate.run()
    for p, g in zip([[5, 6], *prompts, [12], [13]], [a, *got, late[0],
                                                     late[2]]):
        want = solo.generate(p, _cfg(len(g[0][0][0])))
        assert all(t == want for t, _ in g[0])


def test_a_prefill_holds_so_many_tokens(small_model, tokenizer, monkeypatch):
    from luminaai_amd.inference import paged
    monkeypatch.setattr(paged, "PREFILL_TOKENS", 30)
    eng = _engine(small_model, tokenizer)
    assert eng.admissible([(20, 1), (10, 1), (1, 1)]) == 2
    assert eng.admissible([(40, 1), (1, 1)]) == 1
    assert eng.admissible([(5, 3), (5, 1), (5, 1)]) == 2
    assert eng.admissible([(64, 1)]) == eng.admissible([]) == 0
    prompts = [[5] * 20, [6] * 12, [7] * 3]
    outs = eng.run_to_completion(prompts, _cfg(3))
    solo = GenerationEngine(small_model.eval(), tokenizer)
    assert outs == [solo.generate(p, _cfg(3)) for p in prompts]


# ------------------------------------------------------------ on the GPU
@pytest.fixture
def gpu_model(tiny_config):
    from luminaai_amd.models import (DeepSeekTransformer,
                                     config_to_deepseek_config)
    tiny_config.hidden_size, tiny_config.num_heads = 318, 6    # heads of 53
    tiny_config.num_kv_heads = 2
    torch.manual_seed(0)
    m = DeepSeekTransformer(config_to_deepseek_config(tiny_config))
    return m.to("cuda", torch.bfloat16).eval()


@pytest.mark.gpu
def test_gpu_paged_forward_matches_dense(gpu_model):
    """Prefill and decode over pages against dense forwards of the same weights
    in fp32 on the CPU. A value passes about 24 roundings of at most 2^-8 on
    its way to the logits; added up as a random walk they make 5, and the
    bound is three times that."""
    import copy
    ref_model = copy.deepcopy(gpu_model).cpu().float()
    g = torch.Generator().manual_seed(0)
    seqs = [torch.randint(1, 500, (n,), generator=g).cuda()
            for n in (5, 40, 17, 33)]
    at = gpu_model.layers[0].attention
    c = PagedKVCache(2, at.num_kv_heads, at.head_dim, 30, 16, max_seqs=4,
                     max_len=64, device=torch.device("cuda"))
    with torch.no_grad():
        layers, cu = c.prefill([2, 0, 3, 1], [len(s) - 2 for s in seqs])
        out, _, _ = gpu_model(torch.cat([s[:-2] for s in seqs])[None],
                              kv_caches=layers, cu_seqlens=cu)
        got = [[out[0, cu[i]:cu[i + 1]]] for i in range(4)]
        for t in (-2, -1):
            x = torch.stack([s[t] for s in seqs])[:, None]
            out, _, _ = gpu_model(x, kv_caches=c.decode([2, 0, 3, 1]))
            for i in range(4):
                got[i].append(out[i])
        for i, s in enumerate(seqs):
            ref, _, _ = ref_model(s[None].cpu())
            x, y = torch.cat(got[i]).float().cpu(), ref[0]
            assert (x - y).norm() <= 16 * 2 ** -8 * y.norm()


@pytest.mark.gpu
def test_gpu_engine_answers_and_forks(gpu_model, tokenizer):
    prompts = [tokenizer.encode("a first prompt for the engine"),
               tokenizer.encode("b"), tokenizer.encode("the third of them")]
    eng = _engine(gpu_model, tokenizer)
    slots = eng.admit_many(prompts, [_cfg(8, logprobs=2)] * 3)
    fork = eng.fork(slots[0])
    while eng.n_active():
        eng.step()
    assert eng.slots[fork].result == eng.slots[slots[0]].result
    solo = GenerationEngine(gpu_model, tokenizer)
    for p, b in zip(prompts, slots):
        s = eng.slots[b]
        assert len(s.result) == 8
        # greedy: each token is the likeliest at its place, up to what two bf16
        # forwards of different kernels differ by
        score = solo.score([p + s.result], top_k=1)[0]
        for i, e in enumerate(s.logprobs):
            at = len(p) - 1 + i
            assert e["top"][0][0] == e["token"]
            assert score["logprobs"][at] >= \
                score["top_logprobs"][at][0] - 0.25
    _check(eng.cache)
    with pytest.raises(TypeError, match="bf16"):
        _engine(gpu_model.float(), tokenizer)


@pytest.mark.gpu
def test_gpu_packed_training_step(gpu_model):
    """Gradients of a packed batch against those of each sequence alone in fp32
    on the CPU: twice the roundings of a forward (about 50 of 2^-8, 7 as a
    random walk), and three times that as the bound."""
    import copy
    g = torch.Generator().manual_seed(3)
    seqs = [torch.randint(1, 500, (n,), generator=g) for n in (40, 7, 64)]
    w = torch.randn(111, 512, generator=g)
    cu = torch.tensor([0, 40, 47, 111], dtype=torch.int32)

    def grads(m, logits):
        loss = (logits.float() * w.to(logits.device)).sum()
        return torch.autograd.grad(loss, list(m.parameters()))

    ref_model = copy.deepcopy(gpu_model).cpu().float().train()
    b = grads(ref_model, torch.cat([ref_model(s[None])[0][0] for s in seqs]))
    m = gpu_model.train()
    out, _, _ = m(torch.cat(seqs)[None].cuda(), cu_seqlens=cu.cuda())
    for x, y in zip(grads(m, out[0][:, :512]), b):
        assert (x.float().cpu() - y).norm() <= 21 * 2 ** -8 * y.norm()


@pytest.mark.gpu
def test_gpu_paged_moe(tiny_moe_config, tokenizer):
    """Every answer has its length, and its tokens are the likeliest of what the
    model says where it stands."""
    m = _dropping_moe(tiny_moe_config).to("cuda", torch.bfloat16)
    eng = _engine(m, tokenizer)
    # log probabilities are taken before penalties: without one, the greedy token
    # is the likeliest
    cfg = _cfg(8, logprobs=1, repetition_penalty=1.0)
    slots = eng.admit_many(_sequences(12, 33, 40, 25), [cfg] * 4)
    while eng.n_active():
        eng.step()
    for b in slots:
        s = eng.slots[b]
        assert len(s.result) == 8
        for t, e in zip(s.result, s.logprobs):
            assert e["top"][0][0] == t and math.isfinite(e["logprob"])
