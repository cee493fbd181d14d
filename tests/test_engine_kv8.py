"""The serving engine with an 8-bit KV cache, and log probabilities of what it generates, on the CPU."""
import json

import pytest
import torch
from fastapi.testclient import TestClient

from kv8_reference import Cache
from ronn_b200 import Model
from ronn_b200.api.errors import SessionError
from ronn_b200.models.gpt2 import GPT2Config, build_gpt2
from ronn_b200.ops import KV8Cache
from ronn_b200.serving import CachePrecision, EngineConfig, LLMEngine, SamplingParams
from ronn_b200.serving.ops_backend import TorchOps
from ronn_b200.serving.server import create_app


@pytest.fixture(scope="module")
def model():
    return Model.from_graph(build_gpt2(GPT2Config.tiny(n_layer=2, n_embd=128, n_head=2, vocab_size=300, n_positions=128), dtype=torch.float32, seed=1))


def engine(model, **kw):
    cfg = dict(max_num_seqs=4, max_batch_tokens=64, max_model_len=128, num_blocks=32, dtype="fp32", backend="torch")
    cfg.update(kw)
    return LLMEngine(model, EngineConfig(**cfg), device="cpu")


@pytest.mark.parametrize("precision", ["int8", "fp8"])
def test_the_library_backend_stores_what_the_definition_says(precision):
    """Prompts, then tokens one by one; rows without a slot; values of all sizes, some not finite."""
    ops, d = TorchOps(), 64
    cache = KV8Cache.alloc(5, 2, d, precision, device="cpu")
    ref = [Cache(cache.k, cache.k_scale), Cache(cache.v, cache.v_scale)]
    g = torch.Generator().manual_seed(3)
    for slots in ([32, 33, 34, -1, 0, 1], [35, 2], [36, -1], [37, 3], [16, 17, 18]):
        x = (torch.randn(len(slots), 6 * d, generator=g) * torch.exp(2 * torch.randn(len(slots), 1, generator=g))).bfloat16()
        if len(slots) == 3:
            x[1, 2 * d + 5] = float("nan")
            x[2, 5 * d] = float("inf")
        ops.kv8_append(x, 2 * d, 4 * d, torch.tensor(slots, dtype=torch.int32), cache, 2)
        for r, off in zip(ref, (2 * d, 4 * d)):
            r.append(x[:, off:off + 2 * d].reshape(-1, 2, d), slots)
    for codes, scale, r in ((cache.k, cache.k_scale, ref[0]), (cache.v, cache.v_scale, ref[1])):
        live = ~torch.isnan(r.scale[:4])
        assert torch.equal(torch.nan_to_num(scale[:4].double(), nan=-1.0), torch.nan_to_num(r.scale[:4], nan=-1.0))
        assert torch.equal(codes[:4].view(torch.uint8)[live], r.codes[:4].view(torch.uint8)[live])


@pytest.mark.parametrize("precision", ["int8", "fp8"])
def test_generation_keeps_to_the_exact_cache_and_swaps_back_whole(model, precision):
    prompts = [[5 + i] * (9 + 7 * i) for i in range(4)]
    plain = engine(model, kv_cache_dtype=precision)
    assert plain.block_manager.precision == {"int8": CachePrecision.INT8, "fp8": CachePrecision.FP8}[precision]
    assert plain.block_manager.block_bytes == 2 * 2 * (2 * 16 * 64 + 2 * 4)           # layers, k and v, heads: codes and scales
    out = plain.generate(prompts, SamplingParams(max_new_tokens=20))
    assert [len(o) for o in out] == [20] * 4
    # preempted sequences leave with their scales and come back with them
    tight = engine(model, kv_cache_dtype=precision, num_blocks=9, preemption="swap", num_cpu_blocks=32)
    assert tight.generate(prompts, SamplingParams(max_new_tokens=20)) == out
    assert tight.stats()["swapped_blocks"] > 0
    # and a prompt in chunks goes into the same blocks
    assert engine(model, kv_cache_dtype=precision, prefill_chunk=16).generate(prompts, SamplingParams(max_new_tokens=3))[0] == out[0][:3]


def test_a_cache_the_kernels_cannot_hold_is_refused(model):
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        EngineConfig(kv_cache_dtype="int4")
    small = Model.from_graph(build_gpt2(GPT2Config.tiny(n_layer=1, n_embd=64, n_head=2, vocab_size=64, n_positions=32), dtype=torch.float32, seed=0))
    with pytest.raises(SessionError, match="32"):
        engine(small, kv_cache_dtype="int8", max_model_len=32)


def _scores(model, prompt, tokens):
    sess = model.create_session(optimization_level="O0")
    logits = sess.run({"input_ids": torch.tensor([list(prompt) + list(tokens)])})["logits"][0, len(prompt) - 1:-1]
    return torch.log_softmax(logits.double(), -1)


@pytest.mark.parametrize("sampled", [False, True])
def test_log_probabilities_are_the_models(model, sampled):
    """Requests that ask for none, for the token's alone and for alternatives share their steps; penalties and temperature
    change the choice and not the figures."""
    eng = engine(model)
    how = dict(temperature=0.7, repeat_penalty=1.5, seed=4) if sampled else {}
    prompts = [[1, 2, 3], [9] * 20, [4, 4, 7, 8]]
    ids = [eng.add_request(p, SamplingParams(max_new_tokens=6, logprobs=n, **how)) for p, n in zip(prompts, (None, 0, 7))]
    while eng.has_unfinished():
        eng.step()
    plain = engine(model)
    again = [plain.add_request(p, SamplingParams(max_new_tokens=6, **how)) for p in prompts]
    while plain.has_unfinished():
        plain.step()
    reqs = [eng.requests[i] for i in ids]
    assert [r.output_tokens for r in reqs] == [plain.requests[i].output_tokens for i in again]
    assert reqs[0].output_logprobs is None and not eng._logprob_tops
    for r, n, p in ((reqs[1], 0, prompts[1]), (reqs[2], 7, prompts[2])):
        lp = _scores(model, p, r.output_tokens)
        assert [q.token for q in r.output_logprobs] == r.output_tokens
        for q, row in zip(r.output_logprobs, lp):
            assert abs(q.logprob - float(row[q.token])) < 1e-4 and len(q.top) == n
            assert q.rank == 1 + int((row > row[q.token]).sum()) and (sampled or q.rank == 1)
            assert abs(q.entropy - float(-(row.exp() * row).sum())) < 1e-4
            assert [i for i, _ in q.top] == row.argsort(descending=True, stable=True)[:n].tolist()


def test_log_probabilities_are_bounded(model):
    eng = engine(model)
    for n in (-1, 33):
        with pytest.raises(SessionError, match="logprobs"):
            eng.add_request([1], SamplingParams(logprobs=n))


def test_completions_carry_log_probabilities(model):
    from ronn_b200.serving.tokenizer import load_tokenizer
    eng = engine(model, kv_cache_dtype="int8")
    app = create_app(eng, load_tokenizer("bytes", eng.arch.vocab))
    ask = {"prompt_token_ids": [1, 2, 3, 4], "max_tokens": 5, "logprobs": 2}
    with TestClient(app) as c:
        choice = c.post("/v1/completions", json=ask).json()["choices"][0]
        lp = choice["logprobs"]
        assert len(lp["token_logprobs"]) == 5 and all(v <= 0 for v in lp["token_logprobs"]) and lp["ranks"] == [1] * 5
        assert [t[0]["token_id"] for t in lp["top_logprobs"]] == choice["token_ids"] and len(lp["top_logprobs"][0]) == 2
        assert "logprobs" not in c.post("/v1/completions", json={**ask, "logprobs": None}).json()["choices"][0]
        assert c.post("/v1/completions", json={**ask, "logprobs": 99}).status_code == 400
        with c.stream("POST", "/v1/completions", json={**ask, "stream": True}) as s:
            events = [json.loads(l[6:]) for l in s.iter_lines() if l.startswith("data: {")]
        assert [e["logprobs"]["token_id"] for e in events if "token_id" in e] == choice["token_ids"]
        chat = c.post("/v1/chat/completions", json={"messages": [{"role": "user", "content": "hi"}], "max_tokens": 3, "logprobs": True,
                                                    "top_logprobs": 1}).json()["choices"][0]
        assert [p["token_id"] for p in chat["logprobs"]["content"]] == chat["token_ids"]
    app.state.loop.stop()


def test_streamed_chat_carries_log_probabilities(model):
    """Every chunk has those of its own tokens; a request that asks for none gets none."""
    from ronn_b200.serving.tokenizer import load_tokenizer
    eng = engine(model)
    app = create_app(eng, load_tokenizer("bytes", eng.arch.vocab))
    ask = {"messages": [{"role": "user", "content": "hi"}], "max_tokens": 9}
    with TestClient(app) as c:
        whole = c.post("/v1/chat/completions", json={**ask, "logprobs": True, "top_logprobs": 2}).json()["choices"][0]

        def stream(**more):
            with c.stream("POST", "/v1/chat/completions", json={**ask, **more, "stream": True}) as s:
                return [json.loads(l[6:])["choices"][0] for l in s.iter_lines() if l.startswith("data: {")]
        chunks = [x for x in stream(logprobs=True, top_logprobs=2) if "token_ids" in x]
        assert [t for x in chunks for t in x["token_ids"]] == whole["token_ids"]
        assert all([p["token_id"] for p in x["logprobs"]["content"]] == x["token_ids"] for x in chunks)
        got = [p for x in chunks for p in x["logprobs"]["content"]]
        assert [(p["rank"], [t["token_id"] for t in p["top_logprobs"]]) for p in got] == \
            [(p["rank"], [t["token_id"] for t in p["top_logprobs"]]) for p in whole["logprobs"]["content"]]
        assert all(abs(p["logprob"] - w["logprob"]) < 1e-4 for p, w in zip(got, whole["logprobs"]["content"]))
        assert all("logprobs" not in x for x in stream())
    app.state.loop.stop()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_library_backend_gives_log_probabilities_as_they_are_defined(dtype):
    """Rows masked altogether, tokens that are none, NaN and +inf, equal logits: as the operator documents them."""
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(9, 12)
    x[0] = -inf
    x[1, 3:] = -inf
    x[2, 5] = nan
    x[3, 7] = inf
    x[4, [2, 9]] = 4.0
    x[5, 2], x[5, 3] = nan, inf
    x[6, 1], x[6, 2] = -0.0, 0.0
    x[8] = torch.arange(12.0)
    tokens = torch.tensor([4, 2, 5, 1, 9, 3, 2, 12, -1])
    r = TorchOps().token_logprobs(x.to(dtype), tokens, 4)
    assert r.logprob.dtype == r.entropy.dtype == r.top_logprobs.dtype == torch.float32 and r.rank.dtype == r.top_ids.dtype == torch.int32
    assert r.rank.tolist() == [5, 3, 1, 3, 2, 2, 3, 0, 0]
    assert r.top_ids.tolist() == [[0, 1, 2, 3], [0, 1, 2, 3], [5, 0, 1, 2], [7, 0, 1, 2], [2, 9, 0, 1], [2, 3, 0, 1], [0, 1, 2, 3], [0, 1, 2, 3], [11, 10, 9, 8]]
    assert r.logprob[0] == -inf and r.entropy[0] == 0 and bool((r.top_logprobs[0] == -inf).all())
    assert abs(float(r.logprob[1]) + 1.0986123) < 1e-6 and r.top_logprobs[1, 3] == -inf and abs(float(r.entropy[1]) - 1.0986123) < 1e-6
    for row in (2, 3, 5):
        assert torch.isnan(r.logprob[row]) and torch.isnan(r.entropy[row]) and bool(torch.isnan(r.top_logprobs[row]).all())
    assert r.logprob[7] == 0 and r.logprob[8] == 0 and abs(float(r.entropy[7]) - 2.4849066) < 1e-6
    none = TorchOps().token_logprobs(x.to(dtype), None, 4)
    assert bool((none.logprob == 0).all() and (none.rank == 0).all()) and torch.equal(none.top_ids, r.top_ids)


def test_bytes_to_the_host_count_the_log_probabilities(model):
    """Token, log probability, rank and entropy of each request, and the alternatives that the step computed (2 asked for: 5)."""
    eng = engine(model)
    for n in (None, 2, 0):
        eng.add_request([1, 2, 3], SamplingParams(max_new_tokens=4, logprobs=n))
    for _ in range(2):                                               # the prompts, then a decode step
        eng.step()
        assert eng.d2h_bytes_last == 3 * (4 + 12 + 5 * 8)
    plain = engine(model)
    plain.add_request([1, 2, 3], SamplingParams(max_new_tokens=4))
    plain.step()
    assert plain.d2h_bytes_last == 4
