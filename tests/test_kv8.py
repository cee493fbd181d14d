"""The 8-bit cache and the log probabilities on the CPU: refusals of their entry points, index checks, the scale's definition."""
import math

import pytest
import torch

from kv8_reference import Cache, least_scale
from ronn_b200 import ops
from ronn_b200.ops import checks as C


def _cache(blocks=6, kvh=2, d=64, precision="int8"):
    return ops.KV8Cache.alloc(blocks, kvh, d, precision, device="cpu")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


def _q(rows=3, cols=8 * 64, dtype=torch.bfloat16):
    return torch.zeros(rows, cols, dtype=dtype)


def test_cache_shapes_and_types():
    c = _cache(precision="fp8")
    assert c.k.dtype == torch.float8_e4m3fn and c.k.shape == (6, 2, 16, 64) and c.k_scale.shape == (6, 2) and c.num_blocks == 6
    ok = _cache()
    for args in ((ok.k.to(torch.uint8), ok.v.to(torch.uint8), ok.k_scale, ok.v_scale), (ok.k, c.v, ok.k_scale, ok.v_scale),
                 (ok.k[:, :, :8], ok.v[:, :, :8], ok.k_scale, ok.v_scale), (ok.k[..., :32], ok.v[..., :32], ok.k_scale, ok.v_scale),
                 (ok.k, ok.v, ok.k_scale.half(), ok.v_scale), (ok.k, ok.v, ok.k_scale[:5], ok.v_scale),
                 (ok.k.transpose(0, 1), ok.v.transpose(0, 1), ok.k_scale.t(), ok.v_scale.t()), (ok.k[1:], ok.v, ok.k_scale, ok.v_scale)):
        with pytest.raises(ops.OperandError):
            ops.KV8Cache(*args)
    with pytest.raises(ops.OperandError, match="int4"):
        _cache(precision="int4")


def test_append_refusals():
    c, qkv, slots = _cache(), _q(), _i32([0, 1, 2])
    bad = [dict(qkv=_q(dtype=torch.float32)), dict(qkv=_q(cols=8 * 64 - 1)), dict(qkv=_q().t()), dict(qkv=_q(cols=8 * 64 + 3)), dict(qkv=_q()[0]),
           dict(k_off=4 * 64 + 4), dict(v_off=-8), dict(v_off=7 * 64), dict(slots=slots.long()), dict(slots=slots[:2]), dict(heads=3), dict(heads=0),
           dict(slots=_i32([0, 1, 2, 3, 4, 5])[::2]), dict(rotated=_q()), dict(positions=slots[:2], rope_base=1e4),
           dict(positions=slots, rope_base=math.inf), dict(positions=slots, rope_base=1e4, rotated=_q(dtype=torch.float16)),
           dict(positions=slots, rope_base=1e4, rotated=_q(rows=2)), dict(positions=slots, rope_base=1e4, k_off=3 * 64)]
    for change in bad:
        kw = dict(qkv=qkv, k_off=4 * 64, v_off=6 * 64, slots=slots, cache=c, heads=4)
        kw.update(change)
        with pytest.raises(ops.OperandError):
            ops.kv8_append(**kw)
    with pytest.raises(ops.OperandError, match="CUDA device"):       # all right but for where it is
        ops.kv8_append(qkv, 4 * 64, 6 * 64, slots, c, 4)


def test_read_refusals():
    c = _cache()
    for args in ((c, _i32([0]), torch.float32), (c, torch.tensor([0])), (c, _i32([[0, 1]])), (c, _i32([0]))):
        with pytest.raises(ops.OperandError):
            ops.kv8_read(*args)


def test_attention_refusals():
    c, tab, ctx = _cache(), _i32([[0, 1, -1]] * 3), _i32([17, 3, 0])
    good = dict(q=_q(), cache=c, block_tables=tab, ctx_len=ctx, heads=4, max_ctx=32)
    slots = _i32([16, 2, -1])
    for change in (dict(q=_q(dtype=torch.float32)), dict(q=_q(cols=3 * 64)), dict(q=_q(cols=8 * 64 + 4)), dict(block_tables=tab.long()),
                   dict(block_tables=tab[:2]), dict(block_tables=tab.t()), dict(block_tables=tab[0]), dict(ctx_len=ctx[:2]), dict(ctx_len=ctx.long()),
                   dict(bt_row=_i32([0])), dict(heads=5), dict(max_ctx=-1), dict(scale=math.nan), dict(scale=math.inf), dict(rope=(slots, 1e4)),
                   dict(append=(4 * 64, 6 * 64, slots[:2])), dict(append=(4 * 64, 7 * 64, slots)), dict(append=(4 * 64 + 1, 6 * 64, slots)),
                   dict(append=(4 * 64, 6 * 64, slots), rope=(slots, -1.0)), dict(append=(4 * 64, 6 * 64, slots), rope=(slots[:1], 1e4)),
                   dict(block_tables=torch.empty(3, 0, dtype=torch.int32))):
        with pytest.raises(ops.OperandError):
            ops.kv8_attention(**{**good, **change})
    with pytest.raises(ops.OperandError, match="CUDA device"):
        ops.kv8_attention(**good)


def test_chunk_attention_refusals():
    c, tab = _cache(), _i32([[0, 1, -1]] * 2)
    good = dict(q=_q(), q_off=0, cache=c, block_tables=tab, seq_start=_i32([0, 1]), q_len=_i32([1, 2]), kv_len=_i32([5, 20]), max_q_len=2, max_kv_len=20,
                heads=8)
    for change in (dict(q_off=8), dict(q_off=-8), dict(q_off=4, heads=4), dict(q_len=_i32([1])), dict(kv_len=torch.tensor([5, 20])),
                   dict(block_tables=tab[:1]), dict(bt_row=_i32([0])), dict(max_q_len=-1), dict(max_kv_len=-1), dict(heads=7),
                   dict(q=_q(dtype=torch.float32)), dict(seq_start=_i32([[0, 1]])), dict(scale=-math.inf)):
        with pytest.raises(ops.OperandError):
            ops.kv8_prefill_attention(**{**good, **change})
    with pytest.raises(ops.OperandError, match="CUDA device"):
        ops.kv8_prefill_attention(**good)


def test_logprobs_refuse_the_host():
    with pytest.raises(ops.OperandError, match="CUDA device"):
        ops.token_logprobs(torch.zeros(2, 5))


def test_index_check_of_the_append():
    c, qkv = _cache(), _q(5)
    C.kv8_append(qkv, _i32([5, 6, -1, 31, 32]), c.k)
    C.kv8_append(qkv, _i32([15, 16, 17, 64, 33]), c.k)
    for slots in ([0, 1, -1, 2, 3], [3, 2, 1, 0, 16], [0, 0, 16, 32, 48], [7, 16, 8, 32, 48]):
        with pytest.raises(C.IndexCheckError, match="do not stand together"):
            C.kv8_append(qkv, _i32(slots), c.k)
    with pytest.raises(C.IndexCheckError, match=r"slots\[1\] = 96"):
        C.kv8_append(qkv, _i32([0, 96, -1, -1, -1]), c.k)


@pytest.mark.parametrize("code,most", [(torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)])
def test_the_scale_is_the_least_power_of_two_that_holds_the_largest(code, most):
    for amax, e in ((most, 0), (most * (1 + 2 ** -7), 1), (most / 2, -1), (1e-40, -100), (0.0, -100), (most * 2.0 ** 20, 20)):
        assert least_scale(amax, code) == 2.0 ** e


def test_reference_rounds_older_codes_again_when_a_larger_token_joins():
    c = Cache(torch.zeros(1, 1, 16, 2, dtype=torch.int8), torch.zeros(1, 1))
    c.append(torch.tensor([[[1.0, 127.0]]]), [0])
    assert c.scale[0, 0] == 1 and c.codes[0, 0, 0].tolist() == [1, 127]
    c.append(torch.tensor([[[254.0, 3.0]]]), [1])
    assert c.scale[0, 0] == 2 and c.codes[0, 0, :2].tolist() == [[0, 64], [127, 2]]      # 1/2 and 3/2 round to even


def test_chunk_checks_allow_fewer_keys_than_queries():
    start, count, keys = _i32([0, 4]), _i32([4, 3]), _i32([2, 32])
    C.sequences(7, start, count, keys, False, 32, True)
    with pytest.raises(C.IndexCheckError, match="4 queries but only 2 keys"):
        C.sequences(7, start, count, keys, False, 32)
    with pytest.raises(C.IndexCheckError, match="kv_len"):
        C.sequences(7, start, count, _i32([2, 33]), False, 32, True)


def test_columns_that_are_both_rotated_in_place_and_stored_are_refused():
    c, qkv, slots = _cache(), _q(), _i32([0, 1, 2])
    for v_off in (0, 3 * 64, 4 * 64, 5 * 64):
        with pytest.raises(ops.OperandError, match="rotated in place"):
            ops.kv8_append(qkv, 4 * 64, v_off, slots, c, 4, slots, 1e4)
        with pytest.raises(ops.OperandError, match="CUDA device"):
            ops.kv8_append(qkv, 4 * 64, v_off, slots, c, 4, slots, 1e4, _q())
        with pytest.raises(ops.OperandError, match="CUDA device"):
            ops.kv8_append(qkv, 4 * 64, v_off, slots, c, 4)


def test_tables_whose_keys_pass_32_bits_are_refused():
    wide = torch.empty(1, 2 ** 26 + 1, dtype=torch.int32)
    with pytest.raises(ops.OperandError, match="2\\^26"):
        ops.kv8_attention(_q(1), _cache(), wide, _i32([1]), 4, 16)


@pytest.mark.parametrize("base", [10000.0, 500000.0, 1e6, 3.7, 1.0, 1e-30])
@pytest.mark.parametrize("d", [64, 128])
def test_rotary_turns_are_right_to_their_last_bit(base, d):
    """base^(-2j/d) / (2 pi) as 64-bit fractions, against integers: d / 2 is a power of two, so the root is one of square roots,
    and pi is Machin's sum."""
    from fractions import Fraction
    from ronn_b200.ops.kv8 import _turns
    bits = 2000                                                      # base^-64 has fewer zeros behind the point

    def inverse_tangent(x):
        total = term = (1 << bits) // x
        n = 1
        while term:
            term //= -x * x
            n += 2
            total += term // n
            term = 0 if abs(term) <= 1 else term
        return total
    pi = 4 * (4 * inverse_tangent(5) - inverse_tangent(239))
    for j, got in enumerate(_turns(d, base)[0]):
        v = Fraction(base) ** -j
        v = (v.numerator << bits) // v.denominator
        for _ in range((d // 2).bit_length() - 1):
            v = math.isqrt(v << bits)
        want = (v << (bits + 64)) // (2 * pi)                        # in units of 2^-64, with `bits` behind the point
        off = ((got << bits) - want) % (1 << (bits + 64))
        assert min(off, (1 << (bits + 64)) - off) <= (1 << bits) * 51 // 100, (j, base)


def test_rotated_columns_that_overlap_the_activation_elsewhere_are_refused():
    """In place, or apart: a shifted, a differently strided or a partly shared buffer would be read and written at once."""
    c, slots = _cache(), _i32([0, 1, 2])
    buf = torch.zeros(8, 24 * 64, dtype=torch.bfloat16)
    qkv = buf[2:5, 8 * 64:16 * 64]
    flat = buf.view(-1)
    call = lambda rotated, qkv=qkv, n=3: ops.kv8_append(qkv, 4 * 64, 6 * 64, slots[:n], c, 4, slots[:n], 1e4, rotated)
    at = (2 * 24 + 8) * 64                                           # where qkv starts
    for rotated in (buf[1:4, 8 * 64:16 * 64], buf[3:6, 8 * 64:16 * 64], buf[2:5, 9 * 64:17 * 64], buf[2:5, 7 * 64:15 * 64], buf[2:5, 3 * 64:9 * 64 + 8],
                    flat[at:at + 3 * 512].view(3, 512), flat[at - 512:at + 3 * 512 - 512].view(3, 512)):
        with pytest.raises(ops.OperandError, match="overlap"):
            call(rotated)
    apart = (qkv, buf[2:5, :8 * 64], buf[2:5, 16 * 64:], buf[2:5, :6 * 64], buf[5:], _q(),
             buf[2:5, 1 * 64:7 * 64], buf[3:6, 1 * 64:8 * 64])
    for rotated in apart:
        with pytest.raises(ops.OperandError, match="CUDA device"):  # right but for where it is
            call(rotated)
    with pytest.raises(ops.OperandError, match="CUDA device"):       # one row in place, whatever its stride
        call(flat[at:at + 512].view(1, 512), qkv[:1], 1)
    with pytest.raises(ops.OperandError, match="overlap"):
        call(flat[at + 8:at + 520].view(1, 512), qkv[:1], 1)


def test_results_that_overlap_the_queries_are_refused():
    """Query heads are read by other CTAs than the one that writes a result over them."""
    c, tab, three = _cache(), _i32([[0, 1, -1]] * 3), _i32([17, 3, 0])
    buf = torch.zeros(8, 12 * 64, dtype=torch.bfloat16)
    q = buf[2:5, :8 * 64]
    row = lambda out, **kw: ops.kv8_attention(q, c, tab, three, 4, 32, out=out, **kw)
    chunk = lambda out: ops.kv8_prefill_attention(q, 64, c, tab[:1], _i32([0]), _i32([3]), _i32([20]), 3, 20, 4, out=out)
    append = dict(append=(4 * 64, 6 * 64, three))
    for call, bad, good in ((row, (q, buf[1:4, 64:], buf[2:5, 3 * 64:]), (buf[2:5, 4 * 64:], buf[5:], buf[2:5, 8 * 64:])),
                            (lambda out: row(out, **append), (q, buf[2:5, 4 * 64:]), (buf[2:5, 8 * 64:], buf[5:])),
                            (chunk, (q, buf[2:5, 4 * 64:]), (buf[2:5, 5 * 64:], buf[2:5, 8 * 64:], buf[5:]))):
        for out in bad:
            with pytest.raises(ops.OperandError, match="overlap"):
                call(out)
        for out in good:
            with pytest.raises(ops.OperandError, match="CUDA device"):
                call(out)
