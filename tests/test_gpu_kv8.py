"""The 8-bit paged KV cache on the GPU: append, read, decode attention and chunk attention against 64 bits."""
import math

import pytest
import torch

from kv8_reference import Cache, attend, bound, rotate

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def _ops():
    from ronn_b200 import ops
    return ops


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _filled(blocks, kvh, d, code, seed, spread=3.0):
    """A cache whose blocks differ widely in size (scales from 2^-spread to 2^spread), and one garbage byte in 97."""
    g = torch.Generator().manual_seed(seed)
    ops = _ops()
    mk = lambda: torch.randint(0, 256, (blocks, kvh, 16, d), generator=g, dtype=torch.uint8)
    tensors = []
    for _ in range(2):
        c = mk()
        if code == "int8":
            c[c == 128] = 0                                       # -128 is no code
        else:
            c[(c & 127) == 127] = 0                               # nor is NaN
            c = torch.where((c & 127) > 0x60, c & 0x9f, c)        # magnitudes up to 32 most of the time
        tensors.append(c)
    sc = [2.0 ** torch.randint(-int(spread) - 4, int(spread) - 3, (blocks, kvh), generator=g).float() for _ in range(2)]
    cache = ops.KV8Cache(*[t.cuda().view(CODE[code]) for t in tensors], *[s.cuda() for s in sc])
    return cache


def _check_cache(cache, ref_k, ref_v, live=None):
    for mine, codes, ref in ((cache.k_scale, cache.k, ref_k), (cache.v_scale, cache.v, ref_v)):
        assert torch.equal(torch.nan_to_num(mine.cpu().double(), nan=-1.0), torch.nan_to_num(ref.scale, nan=-1.0))
        ok = ~torch.isnan(ref.scale)
        assert torch.equal(codes.cpu().view(torch.uint8)[ok], ref.codes.view(torch.uint8)[ok])


def _activations(tokens, width, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, width, generator=g) * torch.exp(torch.randn(tokens, 1, generator=g))
    return x.to(DT[dtype]).cuda()


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rope", [0.0, 10000.0])
@pytest.mark.parametrize("runs", [[(0, 1)], [(5, 1)], [(0, 16), (3, 40)], [(15, 2), (0, 0), (7, 9), (32, 33)], [(1, 1)] * 37])
def test_append_matches_the_definition(dtype, code, d, rope, runs):
    """Runs are (first position, tokens) of a sequence: from a block's start, its middle and end, over several blocks, none."""
    ops, kvh, heads = _ops(), 3, 6
    need = [(p + n + 15) // 16 for p, n in runs]
    blocks = sum(need) + 3
    cache = _filled(blocks, kvh, d, code, 1)
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(2)).tolist()
    slots, positions, at = [], [], 0
    for (p, n), k in zip(runs, need):
        pages, at = perm[at:at + k], at + k
        slots += [pages[i // 16] * 16 + i % 16 for i in range(p, p + n)]
        positions += [i + 1000 for i in range(p, p + n)]
    tokens = len(slots)
    qkv = _activations(tokens, (heads + 2 * kvh) * d + 8, dtype, 3)
    before = qkv.clone()
    ref = [Cache(cache.k, cache.k_scale), Cache(cache.v, cache.v_scale)]
    k_off, v_off = heads * d, (heads + kvh) * d
    ops.kv8_append(qkv, k_off, v_off, _i32(slots), cache, heads, _i32(positions) if rope else None, rope)
    x = before.cpu()
    k, v = (x[:, o:o + kvh * d].reshape(tokens, kvh, d) for o in (k_off, v_off))
    want = x.clone()
    if rope:
        q = rotate(x[:, :heads * d].reshape(tokens, heads, d), positions, rope)
        k = rotate(k, positions, rope)
        want[:, :heads * d], want[:, k_off:v_off] = q.reshape(tokens, -1), k.reshape(tokens, -1)
    assert torch.equal(qkv.cpu(), want)
    ref[0].append(k, slots)
    ref[1].append(v, slots)
    _check_cache(cache, *ref)


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_append_token_by_token_is_append_at_once_until_the_scale_grows(code):
    """Falling magnitudes: the first token sets the scale, so both ways round once and give the same codes."""
    ops, kvh, d = _ops(), 2, 64
    x = _activations(33, 3 * kvh * d, "bf16", 5) * (2.0 ** -torch.arange(33, device="cuda").float())[:, None].bfloat16()
    x[0], x[16], x[32] = x[0].abs() + 4, x[16].abs() + 4, x[32].abs() + 4
    one, many = (ops.KV8Cache.alloc(4, kvh, d, code) for _ in range(2))
    slots = _i32([(2 - i // 16) * 16 + i % 16 for i in range(33)])
    ops.kv8_append(x, kvh * d, 2 * kvh * d, slots, one, kvh)
    for t in range(33):
        ops.kv8_append(x[t:t + 1], kvh * d, 2 * kvh * d, slots[t:t + 1], many, kvh)
    for a, b in ((one.k, many.k), (one.v, many.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(one.k_scale, many.k_scale) and torch.equal(one.v_scale, many.v_scale)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_append_extremes(dtype, code):
    """Zeros, subnormals, the type's largest values, infinities and NaN; padding rows are no tokens."""
    ops, d, big = _ops(), 64, (1e30 if dtype == "bf16" else 65504.0)
    cache = _filled(6, 1, d, code, 8)
    x = _activations(9, 3 * d, dtype, 9)
    x[0] = 0
    x[1] = torch.finfo(DT[dtype]).smallest_normal / 4
    x[2] = big
    x[3, 70], x[3, 180] = math.inf, 1.0                            # keys of token 3
    x[4, 130] = math.nan                                           # values of token 4
    x[5:8] = math.nan                                              # not cached
    slots = [0, 16, 33, 50, 66, -1, -1, -1, 85]                     # one token to a block: a block stands once in a call
    ref = [Cache(cache.k, cache.k_scale), Cache(cache.v, cache.v_scale)]
    ops.kv8_append(x, d, 2 * d, _i32(slots), cache, 1)
    ref[0].append(x[:, d:2 * d].cpu().reshape(9, 1, d), slots)
    ref[1].append(x[:, 2 * d:].cpu().reshape(9, 1, d), slots)
    _check_cache(cache, *ref)
    assert math.isnan(float(cache.k_scale[3, 0])) and not math.isnan(float(cache.v_scale[3, 0]))
    assert math.isnan(float(cache.v_scale[4, 0])) and not math.isnan(float(cache.k_scale[4, 0]))
    ops.kv8_append(x[8:], d, 2 * d, _i32([48]), cache, 1)           # block 3 begins again
    assert not math.isnan(float(cache.k_scale[3, 0]))


def test_slots_outside_the_cache_are_skipped_and_reported(monkeypatch):
    monkeypatch.delenv("RONN_KERNEL_CHECKS", raising=False)          # the host's checks would refuse it first
    ops, d = _ops(), 64
    cache = _filled(2, 1, d, "int8", 1)
    kept = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    ops.kv8_append(_activations(3, 3 * d, "bf16", 2), d, 2 * d, _i32([32, 33, 2 ** 31 - 1]), cache, 1)
    assert all(torch.equal(a, b) for a, b in zip(kept, (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    with pytest.raises(Exception, match="8-bit KV cache"):
        ops.check_status()
    k, _ = ops.kv8_read(cache, _i32([0, 2, -1]))
    assert not k[1:].any() and k[0].any()
    with pytest.raises(Exception, match="8-bit KV cache"):
        ops.check_status()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [0, 1, 7])
def test_read_gives_the_values(dtype, code, d, n):
    ops = _ops()
    cache = _filled(9, 3, d, code, 4)
    blocks = [(5 * i + 2) % 9 for i in range(n)]
    k, v = ops.kv8_read(cache, _i32(blocks), DT[dtype])
    for got, c, s in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        want = Cache(c, s).values()[torch.tensor(blocks, dtype=torch.long)]
        assert got.shape == (n, 3, 16, d) and torch.equal(got.cpu(), want.to(DT[dtype]))


# ------------------------------------------------------------------------------------------------ attention
def _pages(lens, blocks, seed):
    """Block tables for contexts of these lengths, pages in no order, -1 behind each row's last."""
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = torch.full((len(lens), max(max(lens) + 15, 16) // 16 + 1), -1, dtype=torch.int32), 0
    for i, n in enumerate(lens):
        k = -(-n // 16)
        table[i, :k] = torch.tensor(perm[at:at + k], dtype=torch.int32)
        at += k
    return table


def _compare(out, cache, q, tables, limits, heads, scale=None, p_round=2.0 ** -11, p_floor=2.0 ** -40, kv_round=0.0):
    """q [rows, heads * d]; row r sees limits[r] keys of tables[r]."""
    d = cache.head_dim
    kv, vv = Cache(cache.k, cache.k_scale).values(), Cache(cache.v, cache.v_scale).values()
    sc = 1 / math.sqrt(d) if scale is None else scale
    for r, n in enumerate(limits):
        ref, *about = attend(q[r].cpu().reshape(heads, d), kv, vv, tables[r].tolist(), n, sc)
        got = out[r].cpu().double().reshape(heads, d)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)), r
        off = (got - ref).abs() - bound(ref, *about, q.dtype, d, p_round, p_floor, kv_round)
        assert not (off > 0).any(), (r, n, float(off.max()))


LENS = [[1], [0], [16], [17, 0, 33], [255, 1, 31, 64, 100], [700], [1, 2, 3, 5, 8, 13, 21, 34, 55, 89, 144, 233]]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("heads,kvh,d", [(3, 3, 64), (8, 2, 128), (20, 1, 64), (5, 5, 128), (12, 4, 64), (34, 2, 128)])
@pytest.mark.parametrize("lens", LENS)
def test_decode_attention(dtype, code, heads, kvh, d, lens):
    ops = _ops()
    blocks = sum(-(-n // 16) for n in lens) + 2
    cache, table = _filled(blocks, kvh, d, code, 11), _pages(lens, blocks, 12)
    q = _activations(len(lens), heads * d + 16, dtype, 13) * 0.3
    out = ops.kv8_attention(q, cache, table.cuda(), _i32(lens), heads, max(lens))
    assert out.shape == (len(lens), heads * d)
    _compare(out, cache, q[:, :heads * d], table, lens, heads)
    ops.check_status()


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_decode_rows_that_share_a_table_row_and_write_into_a_wider_buffer(code):
    ops, heads, kvh, d = _ops(), 4, 2, 64
    cache, table = _filled(12, kvh, d, code, 21), _pages([100, 60], 12, 22)
    rows = [1, 0, 0, 1, 0]
    lens = [60, 17, 100, 1, 0]
    q = _activations(5, heads * d, "bf16", 23)
    buf = torch.full((7, heads * d + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    out = ops.kv8_attention(q, cache, table.cuda(), _i32(lens), heads, 100, bt_row=_i32(rows), out=buf, scale=0.05)
    assert out is buf
    _compare(buf[:5, :heads * d], cache, q, table[rows], lens, heads, 0.05)
    assert bool((buf[5:] == 7).all()) and bool((buf[:, heads * d:] == 7).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("heads,kvh,d", [(2, 2, 64), (8, 2, 128), (6, 1, 64)])
@pytest.mark.parametrize("rope", [0.0, 500000.0])
def test_decode_step_appends_and_attends(dtype, code, heads, kvh, d, rope):
    """The append inside the attention call is the append operator's, to the code; padded rows do nothing."""
    ops = _ops()
    lens = [1, 16, 17, 40, 333, 0, 31]
    blocks = sum(-(-n // 16) for n in lens) + 1
    cache, table = _filled(blocks, kvh, d, code, 31), _pages(lens, blocks, 32)
    slots = [int(table[i, (n - 1) // 16]) * 16 + (n - 1) % 16 if n else -1 for i, n in enumerate(lens)]
    positions = [max(n - 1, 0) for n in lens]
    k_off, v_off = heads * d, (heads + kvh) * d
    qkv = _activations(len(lens), (heads + 2 * kvh) * d, dtype, 33)
    kept = qkv.clone()
    twin = ops.KV8Cache(*[t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)])
    out = ops.kv8_attention(qkv, cache, table.cuda(), _i32(lens), heads, 333, append=(k_off, v_off, _i32(slots)),
                            rope=(_i32(positions), rope) if rope else None)
    assert torch.equal(qkv, kept)
    ops.kv8_append(qkv, k_off, v_off, _i32(slots), twin, heads, _i32(positions) if rope else None, rope)
    assert torch.equal(cache.k.view(torch.uint8), twin.k.view(torch.uint8)) and torch.equal(cache.k_scale, twin.k_scale)
    assert torch.equal(cache.v.view(torch.uint8), twin.v.view(torch.uint8)) and torch.equal(cache.v_scale, twin.v_scale)
    q = (qkv if rope else kept)[:, :heads * d]                        # kv8_append rotated it in place
    _compare(out, cache, q, table, lens, heads)
    ops.check_status()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("heads,kvh,d", [(2, 2, 64), (8, 2, 128), (3, 1, 64)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("form", ["direct", "expanded"])
@pytest.mark.parametrize("chunks", [[(1, 1)], [(5, 5), (3, 200), (0, 7), (17, 17)], [(130, 400)], [(33, 20), (4, 0)], [(64, 64), (257, 300)]])
def test_chunk_attention(dtype, code, heads, kvh, d, causal, chunks, form):
    """(queries, keys) of each sequence: whole prompts, tails, no queries, fewer keys than queries, no keys."""
    ops = _ops()
    lens = [k for _, k in chunks]
    blocks = sum(-(-n // 16) for n in lens) + 2
    cache, table = _filled(blocks, kvh, d, code, 41), _pages(lens, blocks, 42)
    starts, at = [], 2
    for n, _ in chunks:
        starts.append(at)
        at += n + 1                                                   # a row between sequences belongs to none
    q = _activations(at + 1, heads * d + 8, dtype, 43) * 0.5
    out = torch.full((at + 1, heads * d), 9.0, dtype=DT[dtype], device="cuda")
    ops.kv8_prefill_attention(q, 8, cache, table.cuda(), _i32(starts), _i32([n for n, _ in chunks]), _i32(lens),
                              max(n for n, _ in chunks), max(lens), heads, causal, out=out, form=form)
    rows, tables, limits = [], [], []
    for i, (n, k) in enumerate(chunks):
        for j in range(n):
            rows.append(starts[i] + j)
            tables.append(table[i])
            limits.append(max(0, k - (n - 1 - j)) if causal else k)
    _compare(out[rows], cache, q[rows][:, 8:8 + heads * d], tables, limits, heads, p_round=torch.finfo(DT[dtype]).eps / 2,
             p_floor=2.0 ** -25 if dtype == "fp16" else 2.0 ** -40)          # long chunks: p itself in the activations' type
    others = [r for r in range(at + 1) if r not in set(rows)]
    assert bool((out[others] == 9).all())
    ops.check_status()


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("tensor", ["k", "v"])
@pytest.mark.parametrize("n", [3, 200])
@pytest.mark.parametrize("form", ["direct", "expanded"])
def test_a_poisoned_block_is_seen_by_those_who_see_it(code, tensor, n, form):
    """Queries in front of the block read numbers, queries behind it NaN; garbage behind the context stays out."""
    ops, heads, kvh, d = _ops(), 4, 2, 64
    keys = n + 40
    blocks = -(-keys // 16) + 1
    cache, table = _filled(blocks, kvh, d, code, 51), _pages([keys], blocks, 52)
    bad = (keys - 2) // 16                                            # logical block of the last keys
    getattr(cache, tensor + "_scale")[int(table[0, bad]), 1] = math.nan
    cache.v.view(torch.uint8)[int(table[0, (keys - 1) // 16]), :, keys % 16 or 16:] = 0x7f
    cache.k.view(torch.uint8)[int(table[0, (keys - 1) // 16]), :, keys % 16 or 16:] = 0x7f
    q = _activations(n, heads * d, "bf16", 53)
    out = ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([0]), _i32([n]), _i32([keys]), n, keys, heads, form=form)
    sees = [keys - (n - 1 - j) > bad * 16 for j in range(n)]
    nan = torch.isnan(out).cpu().reshape(n, heads, d)
    for j in range(n):
        assert bool(nan[j, 2:].all()) == sees[j] and bool(nan[j, 2:].any()) == sees[j] and not nan[j, :2].any()


def test_pages_outside_the_cache_are_left_out_and_reported(monkeypatch):
    monkeypatch.delenv("RONN_KERNEL_CHECKS", raising=False)          # the host's checks would refuse it first
    ops, d = _ops(), 64
    cache = _filled(4, 2, d, "int8", 61)
    table = torch.tensor([[0, 9, 1], [2, 3, -1]], dtype=torch.int32)
    q = _activations(2, 2 * d, "fp16", 62)
    out = ops.kv8_attention(q, cache, table.cuda(), _i32([48, 32]), 2, 48)
    _compare(out, cache, q, torch.tensor([[0, 1, -1], [2, 3, -1]], dtype=torch.int32), [32, 32], 2)
    with pytest.raises(Exception, match="8-bit KV cache"):
        ops.check_status()


def test_expanded_chunks_in_groups_and_bounds_that_do_not_hold(monkeypatch):
    """More contexts than are expanded at a time; sequences that pass the bounds or the buffer are left out and reported."""
    monkeypatch.delenv("RONN_KERNEL_CHECKS", raising=False)          # the host's checks would refuse it first
    ops, heads, kvh, d = _ops(), 8, 8, 128
    keys, n_seq = 16000, 5                                            # 65 MiB of values a sequence: 3 at a time
    blocks = keys // 16
    cache, table = _filled(blocks, kvh, d, "int8", 91), _pages([keys], blocks, 92)
    table = torch.stack([table[0].roll(17 * i)[:blocks].clamp(min=0) for i in range(n_seq)])
    q = _activations(n_seq * 3, heads * d, "bf16", 93) * 0.2
    kv_len = [keys, 77, 0, keys - 5, 1]
    out = ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([3 * i for i in range(n_seq)]), _i32([3] * n_seq), _i32(kv_len), 3, keys, heads,
                                    form="expanded")
    limits = [max(0, kv_len[i // 3] - 2 + i % 3) for i in range(3 * n_seq)]
    _compare(out, cache, q, table.repeat_interleave(3, 0), limits, heads, p_round=2.0 ** -8)
    ops.check_status()
    for start, count, keys_of, form in (([0, 13], [3, 3], [50, 50], "expanded"), ([0, 3], [3, 4], [50, 50], "expanded"), ([0, 3], [3, 3], [50, 99], "expanded"),
                                        ([0, 13], [3, 3], [50, 50], "direct"), ([0, -1], [3, 3], [50, 50], "direct")):
        out = torch.full((15, heads * d), 5.0, dtype=torch.bfloat16, device="cuda")
        ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32(start), _i32(count), _i32(keys_of), 3, 64, heads, out=out, form=form)
        _compare(out[:3], cache, q, table[[0, 0, 0]], [48, 49, 50], heads, p_round=2.0 ** -8)
        assert bool((out[3:] == 5).all())
        with pytest.raises(Exception, match="8-bit KV cache"):
            ops.check_status()


def test_captured_decode_steps_replay_on_new_contents():
    """Two graphs captured with the same cache, replayed in turn on two streams with new contexts in the same buffers."""
    ops, heads, kvh, d = _ops(), 4, 4, 64
    lens = [70, 500]
    blocks = sum(-(-n // 16) for n in lens) + 2
    cache, table = _filled(blocks, kvh, d, "int8", 71), _pages(lens, blocks, 72)
    tab, ctx = table.cuda(), _i32(lens)
    qs = [_activations(2, heads * d, "bf16", 73 + i) for i in range(2)]
    outs, graphs = [], []
    for q in qs:
        ops.kv8_attention(q, cache, tab, ctx, heads, 512)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.kv8_attention(q, cache, tab, ctx, heads, 512))
        graphs.append(g)
    for new in ([70, 500], [3, 499], [0, 17]):
        ctx.copy_(_i32(new))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(5):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for q, o in zip(qs, outs):
            _compare(o, cache, q, table, new, heads)


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_scales_that_are_no_powers_of_two(code):
    """A cache that something else filled: read, attended to, and appended to (its scale stays where it is large enough)."""
    ops, heads, kvh, d = _ops(), 4, 2, 64
    lens = [70, 33]
    cache, table = _filled(8, kvh, d, code, 101), _pages(lens, 8, 102)
    g = torch.Generator().manual_seed(103)
    for s in (cache.k_scale, cache.v_scale):
        s.mul_(1 + torch.rand(8, kvh, generator=g).cuda())
    q = _activations(2, heads * d, "bf16", 104)
    _compare(ops.kv8_attention(q, cache, table.cuda(), _i32(lens), heads, 70), cache, q, table, lens, heads)
    for form in ("direct", "expanded"):
        out = ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([0, 1]), _i32([1, 1]), _i32(lens), 1, 70, heads, form=form)
        # expanded to bf16, values that are no code times a power of two are rounded
        _compare(out, cache, q, table, lens, heads, p_round=2.0 ** -8, kv_round=2.0 ** -8 if form == "expanded" else 0.0)
    at = int(table[0, 4]) * 16 + 6
    old = [t.clone() for t in (cache.k, cache.k_scale)]
    x = _activations(1, 3 * kvh * d, "bf16", 105) * 1e-3
    ops.kv8_append(x, kvh * d, 2 * kvh * d, _i32([at]), cache, kvh)
    assert torch.equal(cache.k_scale, old[1])
    back = cache.k.float()[at // 16, :, 6] * cache.k_scale[at // 16][:, None]
    step = cache.k_scale[at // 16][:, None] * (0.5 if code == "int8" else 0.0)
    want = x[0, kvh * d:2 * kvh * d].float().view(kvh, d)
    assert bool(((back - want).abs() <= step * (1 + 2.0 ** -10) + want.abs() * (0 if code == "int8" else 2.0 ** -4) + cache.k_scale[at // 16][:, None] * 2.0 ** -9).all())


def test_lengths_written_just_before_the_call():
    """An expanded chunk goes by what the stream holds when it runs, captured and replayed with new lengths too."""
    ops, heads, kvh, d = _ops(), 4, 4, 64
    cache, table = _filled(40, kvh, d, "int8", 111), _pages([300, 300], 40, 112)
    q, tab = _activations(64, heads * d, "bf16", 113), table.cuda()
    start, count, keys = _i32([0, 0]), _i32([0, 0]), _i32([0, 0])
    out = torch.zeros(64, heads * d, dtype=torch.bfloat16, device="cuda")
    call = lambda: ops.kv8_prefill_attention(q, 0, cache, tab, start, count, keys, 40, 300, heads, out=out, form="expanded")
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for run in (call, g.replay):
        for s, n, k in (([0, 40], [40, 24], [300, 77]), ([5, 0], [7, 2], [16, 300]), ([0, 30], [30, 0], [0, 8])):
            fresh = [_i32(v) for v in (s, n, k)]
            out.fill_(3.0)
            for dst, src in zip((start, count, keys), fresh):
                dst.copy_(src)
            run()
            rows = [s[i] + j for i in range(2) for j in range(n[i])]
            limits = [max(0, k[i] - (n[i] - 1 - j)) for i in range(2) for j in range(n[i])]
            _compare(out[rows], cache, q[rows], [table[i] for i in range(2) for _ in range(n[i])], limits, heads, p_round=2.0 ** -8)
            assert bool((out[[r for r in range(64) if r not in set(rows)]] == 3).all())
    ops.check_status()


def test_cache_of_more_than_2_31_codes():
    """Pages whose codes start beyond 32-bit offsets."""
    ops, kvh, d = _ops(), 32, 128
    blocks = (2 ** 31) // (kvh * 16 * d) + 40
    cache = ops.KV8Cache.alloc(blocks, kvh, d, "fp8")
    small = _filled(3, kvh, d, "fp8", 81)
    at = [blocks - 1, blocks - 39, 5]
    for src, dst in ((small.k, cache.k), (small.v, cache.v)):
        dst.view(torch.uint8)[at] = src.view(torch.uint8)
    cache.k_scale[at], cache.v_scale[at] = small.k_scale, small.v_scale
    q = _activations(1, kvh * d, "bf16", 82)
    table = torch.tensor([at], dtype=torch.int32)
    out = ops.kv8_attention(q, cache, table.cuda(), _i32([43]), kvh, 43)
    _compare(out, small, q, torch.tensor([[0, 1, 2]]), [43], kvh)
    chunk = ops.kv8_prefill_attention(q.expand(40, -1).contiguous(), 0, cache, table.cuda(), _i32([0]), _i32([40]), _i32([43]), 40, 43, kvh)
    _compare(chunk[39:], small, q, torch.tensor([[0, 1, 2]]), [43], kvh, p_round=2.0 ** -8)
    ops.kv8_append(torch.cat([q, q, q], 1), kvh * d, 2 * kvh * d, _i32([(blocks - 1) * 16]), cache, kvh)
    k, v = ops.kv8_read(cache, _i32([blocks - 1]))
    assert float((k[0, :, 0].reshape(-1).double() - q[0].double()).abs().max()) <= float(q.abs().max()) * 2.0 ** -4
    assert torch.equal(k[:, :, 0], v[:, :, 0])


def test_calls_on_several_streams_share_a_cache():
    """Decode steps of different sequences on different streams, append included, each behind the kernels that made its inputs."""
    ops, heads, kvh, d = _ops(), 8, 4, 64
    lens = [900 + 37 * i for i in range(6)]
    blocks = sum(-(-n // 16) for n in lens) + 1
    cache, table = _filled(blocks, kvh, d, "fp8", 121), _pages(lens, blocks, 122)
    tab = table.cuda()
    rows = [_activations(1, (heads + 2 * kvh) * d, "bf16", 130 + i) for i in range(6)]
    k_off, v_off = heads * d, (heads + kvh) * d
    twin = ops.KV8Cache(*[t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)])
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream() for _ in range(3)]
    for i in range(6):
        with torch.cuda.stream(streams[i % 3]):
            qkv = rows[i] * 0.5
            slot = _i32([int(table[i, (lens[i] - 1) // 16]) * 16 + (lens[i] - 1) % 16])
            outs.append((qkv, slot, ops.kv8_attention(qkv, cache, tab[i:i + 1], _i32([lens[i]]), heads, lens[i], append=(k_off, v_off, slot))))
    torch.cuda.synchronize()
    for i, (qkv, slot, out) in enumerate(outs):
        ops.kv8_append(qkv, k_off, v_off, slot, twin, heads)
        _compare(out, cache, qkv[:, :heads * d], table[i:i + 1], [lens[i]], heads)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in ((cache.k, twin.k), (cache.v, twin.v), (cache.k_scale, twin.k_scale),
                                                                                  (cache.v_scale, twin.v_scale)))


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_a_step_run_twice_leaves_the_same_cache(code):
    """A captured step is run once eagerly and again by its first replay."""
    ops, heads, kvh, d = _ops(), 2, 2, 128
    lens = [20, 48, 33]
    blocks = 9
    cache, table = _filled(blocks, kvh, d, code, 141), _pages(lens, blocks, 142)
    slots = _i32([int(table[i, (n - 1) // 16]) * 16 + (n - 1) % 16 for i, n in enumerate(lens)])
    qkv = _activations(3, 6 * d, "fp16", 143) * 8
    call = lambda: ops.kv8_attention(qkv, cache, table.cuda(), _i32(lens), heads, 48, append=(2 * d, 4 * d, slots), rope=(_i32([n - 1 for n in lens]), 1e4))
    one = call()
    state = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    assert torch.equal(call(), one)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(state, (cache.k, cache.v, cache.k_scale, cache.v_scale)))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales_of_the_scores(scale):
    ops, heads, kvh, d = _ops(), 4, 2, 64
    lens = [50, 77]
    cache, table = _filled(9, kvh, d, "int8", 151), _pages(lens, 9, 152)
    q = _activations(2, heads * d, "bf16", 153) * 0.1
    _compare(ops.kv8_attention(q, cache, table.cuda(), _i32(lens), heads, 77, scale=scale), cache, q, table, lens, heads, scale)
    for form in (None, "direct", "expanded"):                          # a scale that is not positive goes by the codes
        out = ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32([0, 1]), _i32([1, 1]), _i32(lens), 1, 77, heads, scale=scale, form=form)
        _compare(out, cache, q, table, lens, heads, scale, p_round=2.0 ** -8)


def test_rows_of_extreme_queries():
    """Queries with infinities and NaN, zeros and subnormals spoil no other row."""
    ops, heads, kvh, d = _ops(), 2, 2, 64
    lens = [40] * 6
    cache, table = _filled(20, kvh, d, "fp8", 161), _pages(lens, 20, 162)
    q = _activations(6, heads * d, "bf16", 163) * 0.2
    q[0, 3], q[1, 5], q[2] = math.inf, math.nan, 0
    q[3] = 1e-39
    out = ops.kv8_attention(q, cache, table.cuda(), _i32(lens), heads, 40)
    assert torch.isnan(out[0, :d]).all() and torch.isnan(out[1, :d]).all() and not torch.isnan(out[:2, d:]).any() and not torch.isnan(out[2:]).any()
    _compare(out[2:], cache, q[2:].where(q[2:].abs() > 1e-38, torch.zeros_like(q[2:])), table[2:], lens[2:], heads)


def test_a_chunk_with_fewer_keys_than_queries_passes_the_index_checks(monkeypatch):
    """Queries in front of the first key give zeros, with the host's index checks on as without them."""
    monkeypatch.setenv("RONN_KERNEL_CHECKS", "1")
    ops, d = _ops(), 64
    cache = _filled(2, 1, d, "int8", 91)
    out = ops.kv8_prefill_attention(_activations(5, d, "fp16", 92), 0, cache, _i32([[0, 1]]), _i32([0]), _i32([5]), _i32([3]), 5, 3, 1)
    assert (out[:2] == 0).all() and (out[2:] != 0).any(1).all()


def test_a_cache_whose_storage_moved():
    """A cache's calls take its tensors where they are at the call: one set to another storage is read there."""
    ops, d = _ops(), 64
    cache, other = _filled(3, 1, d, "int8", 93), _filled(3, 1, d, "int8", 94)
    want = ops.kv8_read(other, _i32([2, 0]))
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(cache, name).set_(getattr(other, name))
    got = ops.kv8_read(cache, _i32([2, 0]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("heads,kvh,d", [(17, 1, 64), (48, 2, 128), (40, 1, 64)])
@pytest.mark.parametrize("rope", [0.0, 10000.0])
@pytest.mark.parametrize("given", [False, True])
def test_decode_step_appends_once_for_heads_of_several_tiles(code, heads, kvh, d, rope, given):
    """More query heads to a cached head than a tile holds: the new token joins its block once, whose scale it makes grow."""
    ops = _ops()
    lens = [2, 16, 18, 333, 0, 700]
    blocks = sum(-(-n // 16) for n in lens) + 1
    cache, table = _filled(blocks, kvh, d, code, 95), _pages(lens, blocks, 96)
    slots = [int(table[i, (n - 1) // 16]) * 16 + (n - 1) % 16 if n else -1 for i, n in enumerate(lens)]
    positions = [max(n - 1, 0) for n in lens]
    k_off, v_off = heads * d, (heads + kvh) * d
    qkv = _activations(len(lens), (heads + 2 * kvh) * d, "bf16", 97)
    qkv[:, k_off:] *= 16                                              # larger than what most blocks hold
    kept = qkv.clone()
    twin = ops.KV8Cache(*[t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)])
    before = cache.k_scale.clone()
    out = torch.empty(len(lens), heads * d, dtype=torch.bfloat16, device="cuda") if given else None
    got = ops.kv8_attention(qkv, cache, table.cuda(), _i32(lens), heads, 700, append=(k_off, v_off, _i32(slots)), out=out,
                            rope=(_i32(positions), rope) if rope else None)
    assert torch.equal(qkv, kept) and (out is None or got is out) and (cache.k_scale > before).any()
    ops.kv8_append(qkv, k_off, v_off, _i32(slots), twin, heads, _i32(positions) if rope else None, rope)
    for mine, theirs in ((cache.k, twin.k), (cache.v, twin.v), (cache.k_scale, twin.k_scale), (cache.v_scale, twin.v_scale)):
        assert torch.equal(mine.view(torch.uint8), theirs.view(torch.uint8))
    _compare(got, cache, qkv[:, :heads * d], table, lens, heads)
    ops.check_status()


def test_a_loose_bound_of_queries_changes_nothing():
    ops, heads, d = _ops(), 4, 64
    cache = _filled(4, 2, d, "int8", 98)
    args = (_activations(7, heads * d, "bf16", 99), 0, cache, _i32([[0, 1], [2, 3]]), _i32([0, 3]), _i32([3, 4]), _i32([20, 32]))
    for form in ("direct", "expanded"):
        assert torch.equal(ops.kv8_prefill_attention(*args, 4, 32, heads, form=form), ops.kv8_prefill_attention(*args, 2 ** 40, 32, heads, form=form))


@pytest.mark.parametrize("n_seq", [3, 33, 64, 65])
@pytest.mark.parametrize("heads,kvh", [(2, 1), (3, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_expanded_chunks_of_many_sequences(monkeypatch, n_seq, heads, kvh, causal):
    """Each tile of each sequence is worked on once, in whatever order: sequences without queries or keys, of several tiles, with
    fewer keys than queries, and one that passes the bounds and is left out and reported."""
    monkeypatch.delenv("RONN_KERNEL_CHECKS", raising=False)          # the host's checks would refuse the last first
    ops, d = _ops(), 64
    g = torch.Generator().manual_seed(n_seq)
    counts = [(0, 1, 127, 128, 129, 300)[int(torch.randint(6, (1,), generator=g))] for _ in range(n_seq)]
    lens = [int(torch.randint(0, 500, (1,), generator=g)) for _ in range(n_seq)]
    counts[:2], lens[:2], bad = [300, 257], [480, 130], n_seq - 1
    lens[bad] = 600                                                   # behind max_kv_len
    starts = [sum(counts[:i]) for i in range(n_seq)]
    blocks = sum(-(-n // 16) for n in lens) + 1
    cache, table = _filled(blocks, kvh, d, "fp8", 101), _pages(lens, blocks, 102)
    q = _activations(sum(counts), heads * d, "bf16", 103)
    out = torch.full_like(q, 9.0)
    call = lambda form, out: ops.kv8_prefill_attention(q, 0, cache, table.cuda(), _i32(starts), _i32(counts), _i32(lens), 300, 500, heads, causal,
                                                       out=out, form=form)
    call("expanded", out)
    with pytest.raises(Exception, match="8-bit KV cache"):
        ops.check_status()
    rows = [(i, starts[i] + j, max(0, lens[i] - (counts[i] - 1 - j)) if causal else lens[i]) for i in range(n_seq) if i != bad for j in range(counts[i])]
    assert bool((out[starts[bad]:] == 9).all()) and not bool((out[:starts[bad]] == 9).all(1).any())
    some = rows[::max(1, len(rows) // 600)]
    _compare(out[[r for _, r, _ in some]], cache, q[[r for _, r, _ in some]], [table[i] for i, _, _ in some], [n for _, _, n in some], heads,
             p_round=2.0 ** -8)


def test_expanded_chunks_between_products_that_take_tensor_memory():
    """Chunk attention takes all of an SM's tensor memory; products before and behind it in the stream start early and take some."""
    ops, heads, kvh, d, n = _ops(), 16, 16, 64, 700
    lens = [900, 700, 1300]
    cache, table = _filled(sum(-(-k // 16) for k in lens) + 1, kvh, d, "int8", 121), _pages(lens, sum(-(-k // 16) for k in lens) + 1, 122)
    x, w = _activations(3 * n, heads * d, "bf16", 123), _activations(heads * d, heads * d, "bf16", 124) / 32
    tab, start, count, keys = table.cuda(), _i32([0, n, 2 * n]), _i32([n] * 3), _i32(lens)

    def chain():
        y = x
        for _ in range(4):
            q = ops.gemm(y, w)
            y = ops.gemm(ops.kv8_prefill_attention(q, 0, cache, tab, start, count, keys, n, 1300, heads, form="expanded"), w)
        return y
    want = chain()
    torch.cuda.synchronize()
    apart = x
    for _ in range(4):
        q = ops.gemm(apart, w)
        torch.cuda.synchronize()
        o = ops.kv8_prefill_attention(q, 0, cache, tab, start, count, keys, n, 1300, heads, form="expanded")
        torch.cuda.synchronize()
        apart = ops.gemm(o, w)
        torch.cuda.synchronize()
    assert torch.equal(want, apart) and bool(torch.isfinite(want).all())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        again = chain()
    for _ in range(5):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, want)
    ops.check_status()
