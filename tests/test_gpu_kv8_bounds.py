"""Chunks over the 8-bit cache whose pages, table rows or lengths do not hold: both forms answer alike, and report it."""
import pytest
import torch

from test_gpu_kv8 import DT, _activations, _compare, _filled, _i32, _ops, _pages

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def unchecked(monkeypatch):
    monkeypatch.delenv("RONN_KERNEL_CHECKS", raising=False)          # the host's checks would refuse these first


def _reported(ops):
    with pytest.raises(Exception, match="8-bit KV cache"):
        ops.check_status()


def _round(dtype, form):
    """Tolerances of ``bound``: the direct form keeps 2^15 p in fp16, the expanded form p in the activations' type."""
    if form == "direct":
        return dict(p_round=2.0 ** -11, p_floor=2.0 ** -40)
    return dict(p_round=torch.finfo(DT[dtype]).eps / 2, p_floor=2.0 ** -25 if dtype == "fp16" else 2.0 ** -40)


@pytest.mark.parametrize("dtype,code,heads,kvh,d", [("bf16", "int8", 4, 2, 64), ("fp16", "fp8", 3, 1, 128), ("bf16", "fp8", 2, 2, 128)])
@pytest.mark.parametrize("form", ["direct", "expanded"])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_pages_outside_the_cache_are_left_out(dtype, code, heads, kvh, d, form, causal):
    """Absent pages first, last, alone, side by side over a whole step of 128 keys, and all of a context; beside sequences that
    lack none."""
    ops = _ops()
    count, lens = [5, 200, 3, 40], [100, 500, 33, 40]
    blocks = sum(-(-n // 16) for n in lens) + 2
    cache, table = _filled(blocks, kvh, d, code, 201), _pages(lens, blocks, 202)
    bad = {0: [0, 3], 1: [7, *range(16, 24), 31], 2: [0, 1, 2]}
    for i, at in bad.items():
        table[i, at] = torch.tensor([(-1, -2 ** 31, blocks, 2 ** 31 - 1)[k % 4] for k in range(len(at))], dtype=torch.int32)
    starts = [sum(count[:i]) for i in range(4)]
    q = _activations(sum(count), heads * d, dtype, 203) * 0.5
    out = ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32(starts), _i32(count), _i32(lens), 200, 500, heads, causal, form=form)
    tables, limits = [], []
    for i, n in enumerate(count):
        for j in range(n):
            limit = max(0, lens[i] - (n - 1 - j)) if causal else lens[i]
            there = [b for b in range(-(-limit // 16)) if b not in bad.get(i, [])]
            tables.append(table[i, there] if there else table[3])
            limits.append(sum(min(16, limit - 16 * b) for b in there))
    some = [r for r in range(len(limits)) if r < 9 or r % 7 == 0 or r > 200]
    _compare(out[some], cache, q[some], [tables[r] for r in some], [limits[r] for r in some], heads, **_round(dtype, form))
    _reported(ops)
    whole = ops.kv8_prefill_attention(q[208:], 0, cache, table[3:].cuda(), _i32([0]), _i32([40]), _i32([40]), 40, 40, heads, causal, form=form)
    assert torch.equal(whole, out[208:])
    ops.check_status()


@pytest.mark.parametrize("form", ["direct", "expanded"])
@pytest.mark.parametrize("rows", [True, False])
def test_a_table_row_outside_the_table_lists_no_keys(form, rows):
    """Rows of such a sequence are zeros; one without table rows of its own (fewer rows than sequences) is refused."""
    ops, heads, d = _ops(), 4, 64
    cache, table = _filled(9, 2, d, "int8", 211), _pages([60, 50], 9, 212)
    q = _activations(90, heads * d, "bf16", 213)
    if not rows:
        with pytest.raises(ops.OperandError, match="2 rows for 3"):
            ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([0, 30, 60]), _i32([30] * 3), _i32([60, 50, 40]), 30, 60, heads, form=form)
        return
    for bad in (-1, 2, 2 ** 31 - 1, -2 ** 31):
        out = torch.full_like(q, 9.0)
        ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([0, 30, 60]), _i32([30] * 3), _i32([60, 50, 40]), 30, 60, heads, True,
                                  _i32([0, bad, 1]), out=out, form=form)
        assert bool((out[30:60] == 0).all())
        _reported(ops)
        limits = [60 - 29 + j for j in range(30)] + [40 - 29 + j for j in range(30)]
        _compare(torch.cat([out[:30], out[60:]]), cache, torch.cat([q[:30], q[60:]]), [table[0]] * 30 + [table[1]] * 30, limits, heads,
                 **_round("bf16", form))


@pytest.mark.parametrize("form", ["direct", "expanded"])
@pytest.mark.parametrize("max_kv", [96, 1000])
def test_keys_beyond_the_table_are_cut_off(form, max_kv):
    """A context longer than its table's columns list ends with them, for its queries' places too."""
    ops, heads, d = _ops(), 4, 64
    cache = _filled(9, 2, d, "fp8", 221)
    table = torch.tensor([[0, 1, 2, 3, 4, 5], [8, 7, 6, 5, 4, 3]], dtype=torch.int32)
    q = _activations(80, heads * d, "bf16", 223)
    for long in (97, 2 ** 31 - 1):
        out = ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([0, 40]), _i32([40, 40]), _i32([long, 77]), 40, max_kv, heads, form=form)
        _compare(out, cache, q, [table[0]] * 40 + [table[1]] * 40, [96 - 39 + j for j in range(40)] + [77 - 39 + j for j in range(40)], heads,
                 **_round("bf16", form))
        _reported(ops)


def test_single_rows_beyond_the_table_are_cut_off_and_reported():
    ops, heads, d = _ops(), 4, 64
    cache, table = _filled(9, 2, d, "fp8", 225), torch.tensor([[0, 1], [5, 4], [7, 8]], dtype=torch.int32)
    q = _activations(3, heads * d, "bf16", 226)
    for long in (33, 2 ** 31 - 1):
        _compare(ops.kv8_attention(q, cache, table.cuda(), _i32([32, long, 5]), heads, 1000), cache, q, table, [32, 32, 5], heads)
        _reported(ops)


@pytest.mark.parametrize("form", ["direct", "expanded"])
@pytest.mark.parametrize("heads,kvh,d,keys", [(4, 2, 64, 64), (8, 1, 128, 2000)])
@pytest.mark.parametrize("what", ["more queries than max_q_len", "fewer than none", "more keys than max_kv_len", "rows behind the last", "rows in front"])
def test_sequences_that_pass_their_bounds_are_left_out(form, heads, kvh, d, keys, what):
    """Not a row of theirs is written; with few and with many keys (shares of a context that are joined)."""
    ops = _ops()
    blocks = 2 * (-(-keys // 16)) + 10
    cache, table = _filled(blocks, kvh, d, "int8", 231), _pages([keys, keys + 100], blocks, 232)
    q = _activations(30, heads * d, "bf16", 233) * 0.5
    start, count, kv = {"more queries than max_q_len": (5, 8, keys), "fewer than none": (5, -3, keys), "more keys than max_kv_len": (5, 7, keys + 40),
                        "rows behind the last": (24, 7, keys), "rows in front": (-1, 7, keys)}[what]
    out = torch.full_like(q, 9.0)
    ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([0, start]), _i32([5, count]), _i32([keys, kv]), 7, keys, heads, out=out, form=form)
    _reported(ops)
    assert bool((out[5:] == 9).all())
    _compare(out[:5], cache, q[:5], [table[0]] * 5, [keys - 4 + j for j in range(5)], heads, **_round("bf16", form))


@pytest.mark.parametrize("form", ["direct", "expanded"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,query,code,scale", [("bf16", -1e16, 100, 2.0 ** 50), ("bf16", 1e16, 100, 2.0 ** 50), ("bf16", -1e13, 77, 2.0 ** 20),
                                                    ("bf16", 3e4, 77, 2.0 ** 9), ("fp16", 60000, 63, 2.0 ** 10), ("fp16", -60000, 63, 2.0 ** 10)])
def test_scores_of_any_magnitude_count(dtype, query, code, scale, form, causal):
    """All of a row's scores alike, from 1e9 to 1e35 away from 0 on either side: the mean of the values it sees, as for scores
    of 0, to the bit.  Equal keys give equal sums in any order, so that only differences of 0 are left."""
    ops, d, n = _ops(), 64, 150
    cache, table = _filled(20, 1, d, "int8", 241), _pages([300], 20, 242)
    cache.k.fill_(code)
    cache.k_scale.fill_(scale)
    q = torch.full((n, d), query, dtype=DT[dtype], device="cuda")
    out = ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([0]), _i32([n]), _i32([300]), n, 300, 1, causal, form=form)
    zero = ops.kv8_prefill_attention(torch.zeros_like(q), 0, cache, table.cuda(), _i32([0]), _i32([n]), _i32([300]), n, 300, 1, causal, form=form)
    assert torch.equal(out, zero) and bool((out != 0).any(1).all())
    _compare(zero, cache, torch.zeros_like(q), [table[0]] * n, [300 - (n - 1 - j) if causal else 300 for j in range(n)], 1, **_round(dtype, form))
    ops.check_status()


@pytest.mark.parametrize("form", ["direct", "expanded"])
def test_one_key_far_above_the_others(form):
    """Scores some 1e11 apart: the value of the key that lies ahead, whether it comes first, last or in between."""
    ops, d, n = _ops(), 64, 130
    cache, table = _filled(40, 1, d, "int8", 251), _pages([600], 40, 252)
    cache.k.fill_(-100)
    cache.k_scale.fill_(2.0 ** 20)
    q = torch.full((n, d), 1e3, dtype=torch.bfloat16, device="cuda")
    for key in (0, 130, 299, 300, 599):
        cache.k[int(table[0, key // 16]), 0, key % 16] = 100
        out = ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([0]), _i32([n]), _i32([600]), n, 600, 1, False, form=form)
        value = cache.v[int(table[0, key // 16]), 0, key % 16].float() * cache.v_scale[int(table[0, key // 16]), 0]
        assert torch.equal(out.float(), value.expand(n, d))              # codes and scales are exact in bf16
        cache.k[int(table[0, key // 16]), 0, key % 16] = -100
    ops.check_status()
