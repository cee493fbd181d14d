"""token_logprobs on the GPU at the ends of the logits' range: finite logits of any magnitude give numbers."""
import pytest
import torch

from test_gpu_logprobs import DT, _logits, _log_softmax, _reference

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24


def _check(x, tokens, top):
    """Against 64 bits.  With gaps g_j under the row's maximum, S the sum of exp(-g_j) over all but one largest logit and
    n = vocab / 128 + 64 the additions in a chain, in steps of 2^-24:
      a term's gap is rounded up to three times (difference, product with log2 e, log2 e itself), 3 g_j of the term; the
      exponential and the factors of a rescaling are good to 2^-20, 16; a term below 2^-126 may be lost;
      S is off by s = sum_j exp(-g_j) (3 g_j + 16) + n S, and log(1 + S) by s / (1 + S) and its own rounding;
      the sum of g_j exp(-g_j) is off by its terms' share of the same, and by s once more where the rounding of the maximum's
      product with log2 e, half a unit at most, is taken out of it.
    Differences of logits and of logarithms round by half a step of their size each (2^-22 allows eight halves)."""
    from ronn_b200 import ops
    r = ops.token_logprobs(x.cuda(), tokens.cuda(), top)
    rows, vocab = x.shape
    lp, rank, ent, ids, tops = _reference(x, tokens.tolist(), top)
    assert torch.equal(r.rank.cpu().long(), rank) and torch.equal(r.top_ids.cpu().long(), ids)
    v = x.double()
    z = _log_softmax(v)[1]
    gap = v.amax(-1, keepdim=True) - v
    w = torch.exp(-gap)
    others = w.scatter(1, v.argmax(1, keepdim=True), 0.0)
    n = vocab / 128 + 64
    S = others.sum(1)
    s = STEP * ((others * (3 * gap + 16)).sum(1) + n * S) + vocab * 2.0 ** -126
    mean = (w * gap).sum(1) / (1 + S)
    off_mean = (STEP * ((w * gap * (3 * gap + 16)).sum(1) + n * (w * gap).sum(1)) + vocab * 2.0 ** -119 + s + mean * s) / (1 + S)
    for got, want, g in ((r.logprob, lp, gap[torch.arange(rows), tokens]), *((r.top_logprobs[:, k], tops[:, k], gap[torch.arange(rows), ids[:, k]])
                                                                              for k in range(top))):
        got = got.cpu().double()
        assert bool(torch.isfinite(got).all())
        over = (got - want).abs() - s / (1 + S) - 2.0 ** -22 * (g + z + want.abs()) - 2.0 ** -126
        assert not (over > 0).any(), (int(over.argmax()), float(over.max()))
    got = r.entropy.cpu().double()
    over = (got - ent).abs() - s / (1 + S) - off_mean - 2.0 ** -22 * (z + mean) - 2.0 ** -126
    assert bool(torch.isfinite(got).all()) and not (over > 0).any(), (int(over.argmax()), float(over.max()))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("fill", [-1e9, -3e10, -1e10, -1e11, -1e12, -1e15, -1e20, -1e25, -1e29, 5e9, 1e10, 1e15])
def test_masks_and_forced_tokens_of_large_magnitude(dtype, fill):
    """The whole row, all but a late token, the vectors that every warp reads first, nine tenths; and a token forced."""
    vocab = 20011
    x = _logits(7, vocab, "fp32", 11).cpu()
    keep = x.clone()
    x[0] = fill
    x[1] = fill
    x[1, vocab - 5] = 2.0
    x[2, :15000] = fill
    x[3, torch.rand(vocab, generator=torch.Generator().manual_seed(12)) < 0.9] = fill
    x[4, 17], x[5, vocab - 2] = abs(fill), abs(fill)
    x[6] = fill
    x[6, ::3] = fill * (1 + 2.0 ** -6)
    _check(x.to(DT[dtype]), torch.tensor([9, vocab - 5, 16000, int(keep[3].argmax()), 17, 4, 6]), 8)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(60, 20011), (700, 5000), (1, 131073)])
def test_magnitudes_over_the_whole_range(dtype, rows, vocab):
    """Rows around +-10^4 to 10^29, their logits steps of the type apart, so that some share the maximum and others are next to it."""
    g = torch.Generator().manual_seed(rows)
    size = 10.0 ** (4 + 25 * torch.rand(rows, 1, generator=g, dtype=torch.float64)) * torch.where(torch.rand(rows, 1, generator=g) < 0.5, -1.0, 1.0)
    step = torch.finfo(DT[dtype]).eps * torch.randint(0, 40, (rows, vocab), generator=g).double()
    x = (size * (1 + step)).to(DT[dtype])
    x[::3, 5] = 1.0                                                   # an ordinary token beside them
    _check(x, torch.randint(0, vocab, (rows,), generator=g), 3)


def test_fp16_rows_at_the_end_of_the_range():
    """Logits between the type's lowest and -60000, 32 and more apart: a nearly certain token's log probability is the sum of
    the others, whose digits it keeps."""
    vocab = 20011
    x = torch.full((5, vocab), -65504.0)
    for r, m in enumerate((-60000, -60032, -60672, -64000, -65472)):
        x[r, 100 * r + 7] = m
        x[r, 5000:9000] = m - 32
    x = x.half()
    assert x.max(1).values.tolist() == [-60000, -60032, -60672, -64000, -65472]
    _check(x, torch.tensor([7, 107, 207, 307, 407]), 3)
