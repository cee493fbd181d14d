"""The serving engine with an 8-bit KV cache and log probabilities on the GPU: append, attention and log probabilities of real steps."""
import pytest
import torch

from kv8_reference import Cache, attend, bound, rotate

pytestmark = pytest.mark.gpu


def _engine(model, precision, **kw):
    from ronn_b200.serving import EngineConfig, LLMEngine
    cfg = dict(max_num_seqs=8, max_batch_tokens=512, max_model_len=256, num_blocks=128, dtype="bf16", kv_cache_dtype=precision)
    cfg.update(kw)
    return LLMEngine(model, EngineConfig(**cfg), device=torch.device("cuda", 0))


@pytest.fixture(scope="module")
def gpt2():
    from ronn_b200.api.model import Model
    from ronn_b200.models.gpt2 import GPT2Config, build_gpt2
    return Model.from_graph(build_gpt2(GPT2Config.tiny(n_layer=3, n_embd=256, n_head=4, vocab_size=1000, n_positions=256), dtype=torch.bfloat16, seed=5))


@pytest.fixture(scope="module")
def rotary():
    """Rotary embedding, heads of 128 channels."""
    from ronn_b200.api.model import Model
    from ronn_b200.models.bitnet_llama import BitNetConfig, build_bitnet_llama
    return Model.from_graph(build_bitnet_llama(BitNetConfig.tiny(), dtype=torch.bfloat16, seed=3))


def _prompts(vocab):
    g = torch.Generator().manual_seed(0)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (5, 17, 64, 100, 33, 1, 16, 150, 9, 70)]


class _Watched:
    """The engine's operators, with every append and attention on the first layer's cache checked against 64 bits."""

    def __init__(self, ops, cache):
        self.ops, self.cache, self.calls = ops, cache, {"append": 0, "decode": 0, "chunk": 0, "rows": 0}
        self.refs = [Cache(cache.k, cache.k_scale), Cache(cache.v, cache.v_scale)]

    def __getattr__(self, name):
        return getattr(self.ops, name)

    def _stored(self, qkv, k_off, v_off, slots, heads, positions, base):
        """What the call makes of q; the reference takes k and v."""
        d, kvh, t = self.cache.head_dim, self.cache.kv_heads, qkv.shape[0]
        q, k, v = (qkv[:, o:o + n * d].reshape(t, n, d) for o, n in ((0, heads), (k_off, kvh), (v_off, kvh)))
        if base > 0:
            q, k = rotate(q, positions.cpu(), base), rotate(k, positions.cpu(), base)
        for ref, x, codes, scale in ((self.refs[0], k, self.cache.k, self.cache.k_scale), (self.refs[1], v, self.cache.v, self.cache.v_scale)):
            ref.append(x, slots.tolist())
            assert torch.equal(scale.cpu().double(), ref.scale) and torch.equal(codes.cpu().view(torch.uint8), ref.codes.view(torch.uint8))
        return q

    def _attended(self, out, q, tables, limits, p_round):
        kv, vv = (r.values() for r in self.refs)
        for r, n in enumerate(limits):
            ref, *about = attend(q[r], kv, vv, tables[r].tolist(), n, self.cache.head_dim ** -0.5)
            got = out[r].cpu().double().reshape(ref.shape)
            assert bool(((got - ref).abs() <= bound(ref, *about, out.dtype, self.cache.head_dim, p_round)).all())

    def kv8_append(self, qkv, k_off, v_off, slots, cache, heads, positions=None, rope_base=0.0):
        before = qkv.cpu()
        self.ops.kv8_append(qkv, k_off, v_off, slots, cache, heads, positions, rope_base)
        if cache is self.cache:
            self.calls["append"] += 1
            self._stored(before, k_off, v_off, slots, heads, positions, rope_base)

    def kv8_append_attention(self, qkv, k_off, v_off, slots, cache, tables, ctx, heads, max_ctx, positions=None, rope_base=0.0):
        before = qkv.cpu()
        out = self.ops.kv8_append_attention(qkv, k_off, v_off, slots, cache, tables, ctx, heads, max_ctx, positions, rope_base)
        if cache is self.cache:
            self.calls["decode"] += 1
            q = self._stored(before, k_off, v_off, slots, heads, positions, rope_base)
            self._attended(out, q, tables, ctx.tolist(), 2.0 ** -11)
        return out

    def kv8_prefill_attention(self, q, cache, tables, plan, heads, max_ctx):
        out = self.ops.kv8_prefill_attention(q, cache, tables, plan, heads, max_ctx)
        if cache is self.cache:
            self.calls["chunk"] += 1
            for i, (at, n, k) in enumerate(zip(*(plan[f].tolist() for f in ("seq_start", "q_len", "kv_len")))):
                rows = q[at:at + n].cpu()[:, :heads * cache.head_dim].reshape(n, heads, -1)
                self._attended(out[at:at + n], rows, [tables[i]] * n, [k - n + 1 + j for j in range(n)], 2.0 ** -8)
        return out


@pytest.mark.parametrize("precision", ["int8", "fp8"])
@pytest.mark.parametrize("which", ["gpt2", "rotary"])
@pytest.mark.parametrize("prefix", [False, True])
def test_every_append_and_attention_of_a_run(which, precision, prefix, request):
    """Prompts whole and in chunks, prefix hits, decode steps in batches that change: what the engine hands to the operators and
    what they make of it."""
    from ronn_b200.serving import SamplingParams
    eng = _engine(request.getfixturevalue(which), precision, use_cuda_graph=False, prefill_chunk=40, enable_prefix_cache=prefix)
    eng.runner.ops = watched = _Watched(eng.runner.ops, eng.runner.kv8[0])
    head = list(range(40, 80))
    eng.generate([head + [7] * 5], SamplingParams(max_new_tokens=2))
    eng.generate(_prompts(500) + [head + [7 + i] * (3 + i) for i in range(3)], SamplingParams(max_new_tokens=8))
    assert watched.calls["append"] > 3 and watched.calls["decode"] > 8 and watched.calls["chunk"] > 1


@pytest.mark.parametrize("precision", ["int8", "fp8"])
@pytest.mark.parametrize("which", ["gpt2", "rotary"])
def test_replayed_and_eager_steps_write_the_same_codes(which, precision, request):
    from ronn_b200.serving import SamplingParams
    model = request.getfixturevalue(which)
    engs = [_engine(model, precision, use_cuda_graph=g) for g in (True, False)]
    outs = [e.generate(_prompts(500), SamplingParams(max_new_tokens=12)) for e in engs]
    assert outs[0] == outs[1]
    for a, b in zip(engs[0].runner.cache_tensors(), engs[1].runner.cache_tensors()):
        live = slice(0, -1)                                        # the spare block takes padded rows
        assert torch.equal(a[live].view(torch.uint8), b[live].view(torch.uint8))


@pytest.mark.parametrize("base,other,stat,head", [
    (dict(prefill_chunk=16, max_batch_tokens=128), dict(enable_prefix_cache=True), "prefix_hit_blocks", 80),
    (dict(), dict(num_blocks=9, preemption="swap", num_cpu_blocks=64), "swapped_blocks", 4)])
def test_prefix_hits_and_swaps_keep_the_scales(gpt2, base, other, stat, head):
    """Blocks that a later request finds again, and blocks that went to the host and came back, read as they did."""
    from ronn_b200.serving import SamplingParams
    prompts = [list(range(40, 40 + head)) + [7 + i] * (5 + 7 * i) for i in range(4)]
    outs = []
    for kw in (base, {**base, **other}):
        eng = _engine(gpt2, "int8", max_num_seqs=4, **kw)
        outs.append(eng.generate(prompts[:1], SamplingParams(max_new_tokens=2), max_steps=100)
                    + eng.generate(prompts, SamplingParams(max_new_tokens=24), max_steps=500))
    assert eng.stats()[stat] > 0 and [len(o) for o in outs[1]] == [2] + [24] * 4
    # the same codes; what differs is the batch a row shares, which moves a 16-bit rounding here and there
    agree = sum(a == b for x, y in zip(*outs) for a, b in zip(x, y))
    assert outs[0][0] == outs[1][0] and agree >= 88                # of 98


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("sampled", [False, True])
def test_log_probabilities_of_generated_tokens(gpt2, graph, sampled):
    """Asking for them changes no token; each is the log-softmax of an fp32 run over the same context, within what bf16
    activations of three layers leave (2^-5 of a logit's size here)."""
    from ronn_b200.serving import SamplingParams
    how = dict(temperature=0.8, top_k=20, repeat_penalty=1.3, seed=11) if sampled else {}
    prompts = _prompts(1000)[:6]
    plain = _engine(gpt2, "auto", use_cuda_graph=graph).generate(prompts, SamplingParams(max_new_tokens=6, **how))
    eng = _engine(gpt2, "auto", use_cuda_graph=graph)
    ids = [eng.add_request(p, SamplingParams(max_new_tokens=6, logprobs=n, **how)) for p, n in zip(prompts, (0, 3, None, 20, 32, 5))]
    while eng.has_unfinished():
        eng.step()
    assert [eng.requests[i].output_tokens for i in ids] == plain
    sess = gpt2.create_session(optimization_level="O0")
    for i, p, n in zip(ids, prompts, (0, 3, None, 20, 32, 5)):
        r = eng.requests[i]
        if n is None:
            assert r.output_logprobs is None
            continue
        logits = sess.run({"input_ids": torch.tensor([p + r.output_tokens])})["logits"][0, len(p) - 1:-1].float().cpu()
        lp = torch.log_softmax(logits, -1)
        for q, row, raw in zip(r.output_logprobs, lp, logits):
            assert abs(q.logprob - float(row[q.token])) <= 2.0 ** -5 * float(raw.abs().max()) + 2.0 ** -7
            assert len(q.top) == n and [v for _, v in q.top] == sorted((v for _, v in q.top), reverse=True)
            if not sampled:
                assert q.rank == 1 and (n == 0 or q.top[0] == (q.token, pytest.approx(q.logprob, abs=1e-6)))
