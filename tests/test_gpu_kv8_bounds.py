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
