"""token_logprobs on the GPU against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _ops():
    from ronn_b200 import ops
    return ops


def _log_softmax(v):
    """(log p, log of the sum relative to the largest term), with log1p of the other terms' sum: next to a certain token even
    64 bits lose the logarithm of the whole sum."""
    m, at = v.max(-1, keepdim=True)
    z = torch.log1p(torch.exp(v - m).scatter(-1, at, 0.0).sum(-1, keepdim=True))
    return v - m - z + (m - m), z[:, 0] + (m - m)[:, 0]


def _reference(x, tokens, top):
    """x: [rows, vocab] in its own type, on the CPU.  Order: larger first, NaN above all, the lower index among equals."""
    v = x.double()
    lp, z = _log_softmax(v)
    empty = (v == -math.inf).all(-1)
    lp[empty] = -math.inf
    d = torch.where(v == -math.inf, torch.zeros_like(v), v - v.amax(-1, keepdim=True))
    ent = z - (lp.exp() * d).sum(-1)
    ent[torch.isnan(lp).any(-1)] = math.nan
    ent[empty] = 0.0
    key = torch.where(torch.isnan(v), torch.full_like(v, 1e300), v.clamp(max=1e299))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    lps, ranks = [], []
    for r, t in enumerate(tokens):
        given = 0 <= t < x.shape[1]
        lps.append(float(lp[r, t]) if given else 0.0)
        ranks.append(1 + int((order[r] == t).nonzero()) if given else 0)
    return torch.tensor(lps, dtype=torch.float64), torch.tensor(ranks), ent, order[:, :top], lp.gather(1, order[:, :top])


def _close(got, want, gap, z, vocab, what):
    """gap: how far the token's logit lies under the largest; z: log of the sum relative to the largest term.  The difference
    of two logits and the final one round by 2^-24 of their size each (2^-22 allows four).  The sum of the other terms is a
    sum in 32 bits of at most vocab / 128 + 64 terms in any one chain, and exp is good to 2^-20: that relative error of the
    sum moves its logarithm by as much, and by that fraction of it where the sum is small beside 1."""
    rel = (vocab / 128 + 64) * 2.0 ** -24 + 2.0 ** -20
    tol = 2.0 ** -22 * (gap + z + want.abs()) + rel * z.clamp(max=1.0) + 2.0 ** -126
    got, same = got.cpu().double(), torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~same & ~torch.isnan(want)], want[~same & ~torch.isnan(want)]), what
    assert bool(((got - want).abs() <= tol)[same].all()), (what, float(((got - want).abs() - tol)[same].max()))


def _check(logits, tokens, top):
    ops = _ops()
    tok = None if tokens is None else tokens.cuda()
    r = ops.token_logprobs(logits, tok, top)
    rows, vocab = logits.shape
    x = logits.cpu()
    lp, rank, ent, ids, tops = _reference(x, [-1] * rows if tokens is None else tokens.tolist(), top)
    assert r.rank.dtype == torch.int32 and torch.equal(r.rank.cpu().long(), rank)
    assert r.top_ids.dtype == torch.int32 and torch.equal(r.top_ids.cpu().long(), ids)
    v = x.double()
    m = v.amax(-1)
    z = torch.nan_to_num(_log_softmax(v)[1], nan=0.0)
    t = torch.tensor([0] * rows) if tokens is None else tokens.clamp(0, vocab - 1)
    gap = torch.nan_to_num(m - v[torch.arange(rows), t], nan=0.0, posinf=0.0)
    _close(r.logprob, lp, gap, z, vocab, "logprob")
    # entropy: log of the sum and a mean of gaps, each gap good to 2^-24 of itself and weighted like the sum's terms
    d = torch.nan_to_num(v - m[:, None], nan=0.0, neginf=0.0, posinf=0.0)
    p = torch.nan_to_num(torch.softmax(v, -1), nan=0.0)
    rel = (vocab / 128 + 64) * 2.0 ** -24 + 2.0 ** -20
    mean = (p * d.abs()).sum(-1)
    tol = 3 * rel * (mean + z.clamp(max=1.0)) + 2.0 ** -22 * (mean + z) + 2.0 ** -126
    got = r.entropy.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(ent))
    ok = ~torch.isnan(ent)
    assert bool(((got - ent).abs() <= tol)[ok].all()), float(((got - ent).abs() - tol)[ok].max())
    for k in range(top):
        gap = torch.nan_to_num(m - v[torch.arange(rows), ids[:, k]], nan=0.0, posinf=0.0)
        _close(r.top_logprobs[:, k], tops[:, k], gap, z, vocab, f"top {k}")
    return r


def _logits(rows, ld, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, ld, generator=g) * spread).to(DT[dtype]).cuda()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 50257), (3, 2), (5, 31), (2, 256), (7, 257), (4, 1000), (3, 4099), (300, 777), (2, 131073), (1, 600011)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_against_64_bits(dtype, rows, vocab, top, pad):
    x = _logits(rows, vocab + pad, dtype, vocab + rows)[:, :vocab]
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(1))
    tokens[0] = int(x[0].float().argmax())
    _check(x, tokens, min(top, vocab))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_equal_logits_rank_by_index(dtype, vocab):
    """All equal; two values; a plateau on top; the largest values next to one another and strided."""
    x = torch.zeros(6, vocab)
    x[1] = torch.arange(vocab) % 2
    x[2, vocab // 3: vocab // 3 + 20] = 4.0
    x[3] = torch.arange(vocab) / vocab * 10
    x[4] = -torch.arange(vocab) / vocab * 10
    x[5, ::max(1, vocab // 39)] = 7.0
    x[5, 0] = -0.0
    tokens = torch.tensor([vocab - 1, 1, vocab // 3 + 7, vocab - 1, vocab - 1, 3])
    _check(x.to(DT[dtype]).cuda(), tokens, 32)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [33, 20000])
def test_masked_rows_and_special_values(dtype, vocab):
    """Rows masked by -inf or by the type's lowest value, but for one token or altogether; NaN and +inf."""
    low = torch.finfo(DT[dtype]).min
    x = _logits(10, vocab, "fp32", 5).cpu()
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 7] = -3.0
    x[2, 5:] = -math.inf
    x[3] = low
    x[4, 1:] = low
    x[5, 9] = math.nan
    x[6, 4] = math.inf
    x[7, 3], x[7, 30] = -math.inf, 50.0
    x[8, 11], x[8, 12] = math.nan, math.nan
    x[9, 0], x[9, 1] = math.inf, math.inf
    tokens = torch.tensor([3, 7, 30, 2, 0, 9, 4, 3, 11, 1])
    _check(x.to(DT[dtype]).cuda(), tokens, 12)


def test_a_nearly_certain_token_keeps_its_digits():
    x = torch.full((4, 50257), -20.0)
    x[0, 5], x[1, 50256], x[2, 0], x[3, 9] = 0.0, 10.0, 40.0, -8.0
    _check(x.cuda(), torch.tensor([5, 50256, 0, 9]), 2)


def test_tokens_outside_the_vocabulary_are_none():
    x = _logits(5, 100, "fp32", 3)
    _check(x, torch.tensor([-1, 100, 2 ** 31 - 1, 99, 0], dtype=torch.int32), 3)
    r = _check(x, torch.tensor([2 ** 32 + 4, -2 ** 40, 5, 99, 0]), 3)
    assert r.rank[0] == 0 and r.rank[2] > 0
    _check(x, None, 4)


def test_strided_tokens_no_rows_and_refusals():
    ops = _ops()
    x = _logits(4, 50, "bf16", 4)
    t = torch.tensor([[1, 0], [2, 0], [3, 0], [49, 0]], device="cuda")[:, 0]
    a, b = ops.token_logprobs(x, t, 2), ops.token_logprobs(x, t.contiguous(), 2)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    none = ops.token_logprobs(x[:0], t[:0], 2)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 2)
    for args in ((x, t, 33), (x, t, -1), (x[:, :3], t, 4), (x, t[:3], 0), (x.t(), t, 0), (x[0], t[:1], 0), (x.double(), t, 0), (x, t.float(), 0),
                 (x, t.cpu(), 0), (x.cpu(), t, 0)):
        with pytest.raises(ops.OperandError):
            ops.token_logprobs(*args)


def test_rows_of_a_captured_graph_follow_their_inputs():
    ops = _ops()
    x, t = _logits(33, 3001, "fp32", 6), torch.randint(0, 3001, (33,), device="cuda", dtype=torch.int32)
    ops.token_logprobs(x, t, 5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = ops.token_logprobs(x, t, 5)
    for seed in (7, 8):
        x.copy_(_logits(33, 3001, "fp32", seed))
        g.replay()
        want = ops.token_logprobs(x, t, 5)
        assert all(torch.equal(a, b) for a, b in zip(r, want))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,few", [(150, 4), (1, 3), (150, 0)])
def test_the_best_tokens_in_few_threads(dtype, rows, few):
    """Large logits in the vectors of a few threads only (every 256th 16-byte vector), more than there is room for as
    candidates: the alternatives come one by one."""
    vocab, e = 262144, 4 if dtype == "fp32" else 8
    x = torch.randn(rows, vocab // e // 256, 256, e, generator=torch.Generator().manual_seed(rows))
    x[:, :, 3:3 + few] += 40.0
    if few == 0:
        x = torch.round(x)                                            # eleven values: ties across all threads
    _check(x.reshape(rows, vocab).to(DT[dtype]).cuda(), torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(2)), few + 2)


def test_streams_and_many_calls_at_once():
    """Calls on several streams, each on inputs its own stream has just made."""
    ops = _ops()
    streams = [torch.cuda.Stream() for _ in range(4)]
    results = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 4]):
            g = torch.Generator(device="cuda").manual_seed(i)
            x = torch.randn(3 + i, 40001, generator=g, device="cuda") * 3
            t = torch.randint(0, 40001, (3 + i,), generator=g, device="cuda")
            results.append((x, t, ops.token_logprobs(x, t, 7)))
    torch.cuda.synchronize()
    for x, t, r in results:
        again = ops.token_logprobs(x, t, 7)
        assert all(torch.equal(a, b) for a, b in zip(r, again))
    _check(results[5][0], results[5][1].cpu(), 7)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,vocab,pad", [(700, 31, 0), (601, 1000, 3), (650, 5999, 1)])
@pytest.mark.parametrize("top", [0, 5, 31])
def test_many_short_rows(dtype, rows, vocab, pad, top):
    x = _logits(rows, vocab + pad, dtype, rows)[:, :vocab]
    x[5] = 2.0
    x[6, 1:] = -math.inf
    x[7] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(3))
    _check(x, tokens, top)
