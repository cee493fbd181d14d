"""Operators of serving a decoder from an 8-bit KV cache, as cases of known size.

* ``append``: keys and values of new tokens into the paged 8-bit cache (with rotary embedding where the model has it), and
  the blocks they went to read back as values;
* ``decode``: attention of one query row per sequence over that cache, with the row's own append in the same call or without;
* ``chunk``: attention of several new tokens per sequence (prompts read in chunks, prefix hits);
* ``logprobs``: log probability, rank, entropy and the likeliest alternatives of given tokens from logits.

Cache: codes [blocks, kv_heads, 16, head_dim], int8 or e4m3, and one scale for each (block, head), keys and values apart, a
power of two: the least 2^e, e >= -100, with largest magnitude * 2^-e within 127 (int8) or 448 (e4m3).  A block begins when
its slot 0 is written; tokens that join it later can only raise its scale, and the codes below them are rounded again.

A case is a dict of plain values.  ``own`` chooses between the plain form (elementary torch operations) and the framework's
kernels.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CODE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_MOST = {"int8": 127.0, "fp8": 448.0}
_BLOCK = 16
_TABLE = 512                       # smallest number of cache blocks made: a serving process keeps far more than one request's


# ---------------------------------------------------------------------------------------------------- the cases
def _append(name, seqs, new, past, heads, kv_heads, dim, dtype, codes, rope):
    return dict(name=name, op="append", seqs=seqs, new_lo=new[0], new_hi=new[1], past_lo=past[0], past_hi=past[1], heads=heads,
                kv_heads=kv_heads, dim=dim, dtype=dtype, codes=codes, rope=rope)


def _decode(name, rows, ctx, heads, kv_heads, dim, dtype, codes, append, rope):
    return dict(name=name, op="decode", seqs=rows, new_lo=1, new_hi=1, past_lo=ctx[0] - 1, past_hi=ctx[1] - 1, heads=heads,
                kv_heads=kv_heads, dim=dim, dtype=dtype, codes=codes, append=append, rope=rope)


def _chunk(name, seqs, new, past, heads, kv_heads, dim, dtype, codes):
    return dict(name=name, op="chunk", seqs=seqs, new_lo=new[0], new_hi=new[1], past_lo=past[0], past_hi=past[1], heads=heads,
                kv_heads=kv_heads, dim=dim, dtype=dtype, codes=codes, rope=0.0)


def _logprobs(name, rows, vocab, dtype, top, pad=0):
    return dict(name=name, op="logprobs", rows=rows, vocab=vocab, dtype=dtype, top=top, pad=pad)


def listed():
    return [
        # sixteen prompts of a serving step go into the cache of a GPT-2-medium layer; one more chunk of long prompts of a
        # rotary model with grouped heads, most of which end and go on inside a block
        _append("append_prompts_16", 16, (64, 512), (0, 0), 16, 16, 64, "bf16", "int8", 0.0),
        _append("append_chunk_rope_5", 5, (100, 700), (1, 2000), 32, 8, 128, "fp16", "fp8", 10000.0),
        # decode steps: one conversation of odd length (latency), the headline serving batch, the rotary ternary decoder's
        # batch, and a few very long contexts with grouped heads
        _decode("decode_1", 1, (333, 333), 16, 16, 64, "bf16", "int8", True, 0.0),
        _decode("decode_256", 256, (64, 768), 16, 16, 64, "bf16", "int8", True, 0.0),
        _decode("decode_rope_128", 128, (41, 577), 20, 20, 128, "bf16", "fp8", True, 10000.0),
        _decode("decode_long_gqa_3", 3, (20011, 65536), 32, 8, 128, "fp16", "fp8", False, 0.0),
        # several new tokens per sequence: short tails behind prefix hits, and chunks of long prompts
        _chunk("chunk_tails_9", 9, (1, 24), (200, 1500), 12, 12, 64, "fp16", "int8"),
        _chunk("chunk_prompts_3", 3, (501, 1024), (700, 4000), 32, 8, 128, "bf16", "fp8"),
        # what a request that asks for log probabilities is answered with: one token, the serving batch (logits with the row
        # stride the engine gives them), every position of scored documents, a small batch with many alternatives
        _logprobs("logprobs_1", 1, 50257, "fp32", 5, 7),
        _logprobs("logprobs_256", 256, 50257, "fp32", 5, 7),
        _logprobs("logprobs_scores_4662", 4662, 50257, "bf16", 0),
        _logprobs("logprobs_top20_37", 37, 32000, "fp16", 20),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "chunk", "logprobs"])
    dtype = rng.choice(["bf16", "fp16"])
    codes = rng.choice(["int8", "fp8"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16, 20]) if dim == 64 else rng.choice([1, 2, 4, 8, 20])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 8] if kv_heads <= 4 else [1, 1, 2])
    rope = rng.choice([0.0, 10000.0])
    width = kv_heads * dim
    if op == "append":
        seqs = _log_int(rng, 1, 24)
        hi = _log_int(rng, 1, max(2, min(1000, 8000000 // (seqs * width))))
        past = _log_int(rng, 1, 3000) if rng.random() < 0.6 else 0
        case = _append("", seqs, (max(1, hi // 3), hi), (past // 3, past), heads, kv_heads, dim, dtype, codes, rope)
    elif op == "decode":
        seqs = _log_int(rng, 1, 256)
        hi = _log_int(rng, 2, max(3, min(60000, 180000000 // (seqs * width))))
        append = rng.random() < 0.5
        case = _decode("", seqs, (max(1, hi // rng.choice([1, 3, 9])), hi), heads, kv_heads, dim, dtype, codes, append,
                       rope if append else 0.0)
    elif op == "chunk":
        seqs = _log_int(rng, 1, 16)
        new = _log_int(rng, 2, 1000)
        past = _log_int(rng, 1, 4000)
        seqs = max(1, min(seqs, int(18e9 // (heads * dim * new * (new + past)))))
        case = _chunk("", seqs, (max(1, new // 3), new), (past // 3, past), heads, kv_heads, dim, dtype, codes)
    else:
        vocab = _log_int(rng, 1000, 130000)
        rows = _log_int(rng, 1, max(1, min(4000, 200000000 // vocab)))
        case = _logprobs("", rows, vocab, rng.choice(["fp32", "bf16", "fp16"]), rng.choice([0, 1, 5, 20]), rng.choice([0, 0, 1, 7, 8]))
    del case["name"]
    return case


def _spread(lo, hi, n, phase=0.5):
    """n whole numbers over [lo, hi] in a scattered order, the largest among them; the same for every seed."""
    v = [lo + int((hi - lo) * ((i * 0.6180339887498949 + phase) % 1.0) + 0.5) for i in range(n)]
    v[n // 2] = hi
    return v


def _lengths(case):
    """(new tokens, tokens cached before them) of each sequence."""
    return _spread(case["new_lo"], case["new_hi"], case["seqs"]), _spread(case["past_lo"], case["past_hi"], case["seqs"], 0.1)


# ---------------------------------------------------------------------------------------------------- inputs
def _states(gen, shape):
    """Keys or values [..., tokens, channels] as a decoder has them: some channels several times the others, and tokens
    that differ in size."""
    d = shape[-1]
    gain = torch.ones(shape[1], 1, d, device="cuda")
    gain[:, :, 3::29] = 5.0
    size = torch.exp(0.3 * torch.randn(shape[0], shape[1], shape[2], 1, generator=gen, device="cuda"))
    return torch.randn(shape, generator=gen, device="cuda") * gain * size


def _least_scale(amax, codes):
    """The least power of two 2^e, e >= -100, with amax * 2^-e within the codes' largest value."""
    frac, exp = torch.frexp(amax)                                      # amax = frac * 2^exp, frac in [0.5, 1)
    top_frac, top_exp = math.frexp(_MOST[codes])
    e = exp - top_exp + (frac > top_frac).to(exp.dtype)
    e = torch.where(amax > 0, e, torch.full_like(e, -100)).clamp(min=-100)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _to_codes(x, codes):
    return torch.round(x).clamp(-127, 127).to(torch.int8) if codes == "int8" else x.to(torch.float8_e4m3fn)


def _filled(gen, blocks, kv_heads, dim, codes):
    """A cache in use: every block holds sixteen tokens."""
    c = torch.empty(blocks, kv_heads, _BLOCK, dim, dtype=_CODE[codes], device="cuda")
    s = torch.empty(blocks, kv_heads, device="cuda")
    for b in range(0, blocks, 4096):
        x = _states(gen, (min(4096, blocks - b), kv_heads, _BLOCK, dim))
        sc = _least_scale(x.abs().amax((2, 3)), codes)
        c[b:b + 4096] = _to_codes(x / sc[:, :, None, None], codes)
        s[b:b + 4096] = sc
    return c, s


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "logprobs":
        dt, ld = _DT[case["dtype"]], case["vocab"] + case["pad"]
        x = torch.empty(case["rows"], ld, dtype=dt, device="cuda")
        for r in range(0, case["rows"], 256):
            # next-token scores: a few tokens lead clearly
            g = torch.randn(min(256, case["rows"] - r), ld, generator=gen, device="cuda")
            x[r:r + 256] = (1.7 * g + 0.35 * g.abs().pow(3) * g.sign()).to(dt)
        logits = x[:, :case["vocab"]]
        tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device="cuda", dtype=torch.int32)
        best = logits.float().argmax(1).to(torch.int32)                                  # most given tokens are likely ones
        pick = torch.rand(case["rows"], generator=gen, device="cuda") < 0.6
        return dict(case=case, logits=logits, tokens=torch.where(pick, best, tokens))
    dt, h, kvh, d = _DT[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    new, past = _lengths(case)
    need = [-(-(n + p) // _BLOCK) for n, p in zip(new, past)]
    blocks = max(sum(need) + 8, _TABLE)
    where = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()     # pages in no order
    pages, at = [], 0
    for n in need:
        pages.append(where[at:at + n])
        at += n
    table = torch.full((len(need), max(need) + 1), -1, dtype=torch.int32)
    for i, p in enumerate(pages):
        table[i, :len(p)] = torch.tensor(p)
    kc, ks = _filled(gen, blocks, kvh, d, case["codes"])
    vc, vs = _filled(gen, blocks, kvh, d, case["codes"])
    tokens = sum(new)
    qkv = torch.randn(tokens, (h + 2 * kvh) * d, generator=gen, device="cuda")
    qkv[:, h * d:] = _states(gen, (1, 2 * kvh, tokens, d))[0].transpose(0, 1).reshape(tokens, 2 * kvh * d)
    starts = [sum(new[:i]) for i in range(len(new))]
    positions = [p + j for n, p in zip(new, past) for j in range(n)]
    item = [i for i, n in enumerate(new) for _ in range(n)]
    st = dict(case=case, qkv=qkv.to(dt), k=kc, v=vc, k_scale=ks, v_scale=vs, table=table.cuda(), positions=_int(positions),
              slots=_int([pages[i][p // _BLOCK] * _BLOCK + p % _BLOCK for i, p in zip(item, positions)]),
              ctx=_int([n + p for n, p in zip(new, past)]), starts=_int(starts), new=_int(new),
              longest=max(n + p for n, p in zip(new, past)), new_lens=new, past_lens=past)
    # the blocks that this call's tokens go to, and for each token which of them is its own
    first = [p // _BLOCK for p in past]
    last = [(n + p - 1) // _BLOCK for n, p in zip(new, past)]
    st["touched"] = _int([pages[i][b] for i in range(len(new)) for b in range(first[i], last[i] + 1)])
    base = [sum(last[j] - first[j] + 1 for j in range(i)) for i in range(len(new))]
    st["token_touched"] = _int([base[i] + p // _BLOCK - first[i] for i, p in zip(item, positions)]).long()
    if case["op"] == "append" and case["rope"]:
        st["rotated"] = torch.zeros_like(st["qkv"])
    if own:
        from ronn_b200 import ops
        st["cache"] = ops.KV8Cache(kc, vc, ks, vs)
    return st


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)(case["op"], case, state)


def _run_own(op, case, st):
    from ronn_b200 import ops
    if op == "logprobs":
        r = ops.token_logprobs(st["logits"], st["tokens"], top=case["top"])
        return {"logprob": r.logprob, "rank": r.rank, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    h, kvh, d, cache = case["heads"], case["kv_heads"], case["dim"], st["cache"]
    k_off, v_off = h * d, (h + kvh) * d
    if op == "append":
        rope = dict(positions=st["positions"], rope_base=case["rope"], rotated=st["rotated"]) if case["rope"] else {}
        ops.kv8_append(st["qkv"], k_off, v_off, st["slots"], cache, h, **rope)
        k, v = ops.kv8_read(cache, st["touched"], st["qkv"].dtype)
        return {"k": k, "v": v, **({"rotated": st["rotated"][:, :v_off]} if case["rope"] else {})}
    if op == "decode":
        out = ops.kv8_attention(st["qkv"], cache, st["table"], st["ctx"], h, st["longest"],
                                append=(k_off, v_off, st["slots"]) if case["append"] else None,
                                rope=(st["positions"], case["rope"]) if case["rope"] else None)
        if not case["append"]:
            return {"out": out}
        k, v = ops.kv8_read(cache, st["touched"], st["qkv"].dtype)
        return {"out": out, "k": k, "v": v}
    return {"out": ops.kv8_prefill_attention(st["qkv"], 0, cache, st["table"], st["starts"], st["new"], st["ctx"], max(st["new_lens"]),
                                             st["longest"], h)}


def _rotate(x, positions, base):
    """Rotary embedding of [tokens, heads, d]: channels (j, j + d / 2) turn by position * base^(-2 j / d)."""
    d = x.shape[-1]
    j = torch.arange(d // 2, device=x.device, dtype=torch.float64)
    angle = positions.double()[:, None, None] * torch.pow(torch.tensor(base, dtype=torch.float64, device=x.device), -2.0 * j / d)
    c, s = angle.cos(), angle.sin()
    a, b = x[..., :d // 2].double(), x[..., d // 2:].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


def _store(x, cache, scales, st, codes):
    """x: [tokens, kv_heads, d] in fp32 into the blocks this call touches."""
    touched, own_block, off = st["touched"].long(), st["token_touched"], (st["slots"] % _BLOCK).long()
    n = touched.numel()
    begins = torch.full((n,), _BLOCK, dtype=torch.long, device=x.device).scatter_reduce(0, own_block, off, "amin")
    amax = torch.zeros(n, x.shape[1], device=x.device)
    amax = amax.scatter_reduce(0, own_block[:, None].expand(-1, x.shape[1]), x.abs().amax(2), "amax")
    before = torch.where((begins == 0)[:, None], torch.zeros_like(amax), scales[touched])
    after = torch.maximum(before, _least_scale(amax, codes))
    raw = cache.view(torch.uint8)
    kept = raw[touched]
    again = _to_codes(kept.view(cache.dtype).float() * (before / after)[:, :, None, None], codes).view(torch.uint8)
    older = torch.arange(_BLOCK, device=x.device)[None, :] < begins[:, None]
    block = torch.where(older[:, None, :, None], again, kept)
    block[own_block, :, off] = _to_codes(x / after[own_block][:, :, None], codes).view(torch.uint8)
    raw[touched] = block
    scales[touched] = after


def _values(cache, scales, blocks):
    b = blocks.long()
    return cache.view(torch.uint8)[b].view(cache.dtype).float() * scales[b][:, :, None, None]


def _attend(q, k, v, seen):
    """q [kv_heads, group, queries, d], k and v [kv_heads, keys, d], seen [queries, keys] -> [kv_heads, group, queries, d]"""
    s = torch.matmul(q, k.transpose(-1, -2)[:, None]) * (1.0 / math.sqrt(q.shape[-1]))
    s = torch.where(seen, s, torch.full_like(s, float("-inf")))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return torch.matmul(p, v[:, None]) / p.sum(-1, keepdim=True)


def _run_plain(op, case, st):
    if op == "logprobs":
        return _logprobs_plain(st["logits"], st["tokens"], case["top"])
    h, kvh, d, codes = case["heads"], case["kv_heads"], case["dim"], case["codes"]
    qkv, t = st["qkv"], st["qkv"].shape[0]
    dt = qkv.dtype
    q = qkv[:, :h * d].view(t, h, d)
    k = qkv[:, h * d:(h + kvh) * d].view(t, kvh, d)
    v = qkv[:, (h + kvh) * d:].view(t, kvh, d)
    if case["rope"]:
        q, k = _rotate(q, st["positions"], case["rope"]), _rotate(k, st["positions"], case["rope"])
    if op == "append" or (op == "decode" and case["append"]):
        _store(k.float(), st["k"], st["k_scale"], st, codes)
        _store(v.float(), st["v"], st["v_scale"], st, codes)
        new = {"k": _values(st["k"], st["k_scale"], st["touched"]).to(dt), "v": _values(st["v"], st["v_scale"], st["touched"]).to(dt)}
        if op == "append":
            if case["rope"]:
                new["rotated"] = torch.cat([q.reshape(t, h * d), k.reshape(t, kvh * d)], 1)
            return new
    else:
        new = {}
    out, at = torch.zeros(t, h * d, dtype=dt, device="cuda"), 0
    for i, (n, past) in enumerate(zip(st["new_lens"], st["past_lens"])):
        ctx = n + past
        pages = st["table"][i, :-(-ctx // _BLOCK)]
        ki = _values(st["k"], st["k_scale"], pages).transpose(0, 1).reshape(kvh, -1, d)[:, :ctx]
        vi = _values(st["v"], st["v_scale"], pages).transpose(0, 1).reshape(kvh, -1, d)[:, :ctx]
        qi = q[at:at + n].float().view(n, kvh, h // kvh, d).permute(1, 2, 0, 3)
        seen = torch.arange(ctx, device="cuda")[None, :] <= torch.arange(past, ctx, device="cuda")[:, None]
        out[at:at + n] = _attend(qi, ki, vi, seen).permute(2, 0, 1, 3).reshape(n, h * d).to(dt)
        at += n
    return {"out": out, **new}


def _logprobs_plain(logits, tokens, top):
    parts = []
    for r in range(0, logits.shape[0], 512):
        x, t = logits[r:r + 512].float(), tokens[r:r + 512].long()[:, None]
        m = x.amax(1, keepdim=True)
        e = torch.exp(x - m)
        z = e.sum(1, keepdim=True, dtype=torch.float64)              # next to 1 where one token leads: 32 bits lose its logarithm
        chosen = x.gather(1, t)
        ahead = (x > chosen) | ((x == chosen) & (torch.arange(x.shape[1], device=x.device)[None, :] < t))
        lead = torch.where(e > 0, x - m, torch.zeros_like(x))
        entropy = torch.log(z) - (e * lead).sum(1, keepdim=True, dtype=torch.float64) / z
        # stable: among equals the lowest index comes first
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top] if top else torch.empty(x.shape[0], 0, dtype=torch.long, device=x.device)
        parts.append((((chosen - m).double() - torch.log(z))[:, 0].float(), ahead.sum(1).to(torch.int32) + 1, entropy[:, 0].float(),
                      order.to(torch.int32), ((x.gather(1, order) - m).double() - torch.log(z)).float()))
    cols = [torch.cat(c) for c in zip(*parts)]
    return dict(zip(("logprob", "rank", "entropy", "top_ids", "top_logprobs"), cols))


# ---------------------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "logprobs":
        return _logprobs64(st["logits"], st["tokens"], case["top"])
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    qkv = st["qkv"].double().view(-1, h + 2 * kvh, d)
    if case["rope"]:
        # channel pairs as complex numbers, turned by exp(i position theta_j); stored in the activations' type
        theta = torch.exp(torch.arange(d // 2, device="cuda", dtype=torch.float64) * (-2.0 / d * math.log(case["rope"])))
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), st["positions"].double()[:, None] * theta)
        z = torch.complex(qkv[:, :h + kvh, :d // 2], qkv[:, :h + kvh, d // 2:]) * turn[:, None]
        qkv = torch.cat([torch.cat([z.real, z.imag], -1).to(st["qkv"].dtype).double(), qkv[:, h + kvh:]], 1)
    result = {}
    if case["op"] == "append" or case.get("append"):
        result["k"] = _blocks64(st, st["k"], st["k_scale"], qkv[:, h:h + kvh], case["codes"])
        result["v"] = _blocks64(st, st["v"], st["v_scale"], qkv[:, h + kvh:], case["codes"])
        if case["op"] == "append":
            if case["rope"]:
                result["rotated"] = qkv[:, :h + kvh].reshape(-1, (h + kvh) * d)
            return result
    out, at = [], 0
    for i, (n, past) in enumerate(zip(st["new_lens"], st["past_lens"])):
        pages = st["table"][i, :-(-(n + past) // _BLOCK)].long()
        ki, vi = _values64(st["k"], st["k_scale"], pages), _values64(st["v"], st["v_scale"], pages)
        rows = []
        for g in range(kvh):
            kg, vg = ki[:, g].reshape(-1, d)[:n + past], vi[:, g].reshape(-1, d)[:n + past]
            q = qkv[at:at + n, g * (h // kvh):(g + 1) * (h // kvh)]                         # [n, group, d]
            s = torch.einsum("ngd,kd->gnk", q, kg) / d ** 0.5
            late = torch.arange(n + past, device="cuda")[None, :] > torch.arange(n, device="cuda")[:, None] + past
            rows.append(torch.einsum("gnk,kd->ngd", torch.softmax(s.masked_fill(late, float("-inf")), -1), vg))
        out.append(torch.cat(rows, 1).reshape(n, h * d))
        at += n
    return {"out": torch.cat(out), **result}


def _values64(cache, scales, pages):
    return cache.view(torch.uint8)[pages].view(cache.dtype).double() * scales[pages].double()[:, :, None, None]


def _blocks64(st, cache, scales, x, codes):
    """Values of the touched blocks after this call's tokens x [tokens, kv_heads, d] have joined them, block by block; the
    codes and scales in ``st`` are brought up to date, for the attention that reads them."""
    values, slots, owner = [], st["slots"].tolist(), st["token_touched"].tolist()
    members = {}
    for t, b in enumerate(owner):
        members.setdefault(b, []).append(t)
    raw = cache.view(torch.uint8)
    for b, page in enumerate(st["touched"].tolist()):
        ts = members[b]
        lo = min(slots[t] % _BLOCK for t in ts)
        new = x[ts[0]:ts[-1] + 1].transpose(0, 1)                                            # [kv_heads, new, d]
        need = torch.ceil(torch.log2(new.abs().amax((1, 2)).clamp(min=2.0 ** -120) / _MOST[codes]) - 1e-9).clamp(min=-100)
        need = need + (new.abs().amax((1, 2)) > _MOST[codes] * torch.exp2(need)).double()
        old = scales[page].double()
        least = ((need.long() + 1023) << 52).view(torch.float64)
        scale = least if lo == 0 else torch.maximum(least, old)
        held = raw[page].view(cache.dtype).double() * old[:, None, None]
        held[:, lo:lo + len(ts)] = new
        # everything but the codes from `lo + len` on is rounded to the block's scale; those stay what they were
        c = held / scale[:, None, None]
        c = torch.round(c).clamp(-127, 127).to(torch.int8) if codes == "int8" else c.float().to(torch.float8_e4m3fn)
        c = c.view(torch.uint8)
        c[:, lo + len(ts):] = raw[page][:, lo + len(ts):]
        raw[page], scales[page] = c, scale.float()
        values.append(c.view(cache.dtype).double() * scale[:, None, None])
    return torch.stack(values)


def _logprobs64(logits, tokens, top):
    out = {k: [] for k in ("logprob", "rank", "entropy", "top_ids", "top_logprobs")}
    for r in range(0, logits.shape[0], 256):
        raw = logits[r:r + 256]
        lp = torch.log_softmax(raw.double(), -1)
        t = tokens[r:r + 256].long()
        value = raw[torch.arange(raw.shape[0], device="cuda"), t]
        below = torch.arange(raw.shape[1], device="cuda") < t[:, None]
        out["logprob"].append(lp[torch.arange(raw.shape[0], device="cuda"), t])
        out["rank"].append(1 + ((raw > value[:, None]).sum(1) + ((raw == value[:, None]) & below).sum(1)).int())
        out["entropy"].append(-(lp.exp() * lp).sum(1))
        left = raw.double()
        ids = []
        for _ in range(top):
            most = left.amax(1, keepdim=True)
            at = torch.where(left == most, torch.arange(raw.shape[1], device="cuda"), raw.shape[1]).amin(1)
            ids.append(at.int())
            left[torch.arange(raw.shape[0], device="cuda"), at] = float("-inf")
        ids = torch.stack(ids, 1) if ids else torch.empty(raw.shape[0], 0, dtype=torch.int32, device="cuda")
        out["top_ids"].append(ids)
        out["top_logprobs"].append(lp.gather(1, ids.long()))
    return {k: torch.cat(v) for k, v in out.items()}


# ---------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    if case["op"] == "logprobs":
        rows, size = case["rows"], {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
        return {"bytes": float(rows) * (case["vocab"] * size + 16 + 8 * case["top"]), "flops": 5.0 * rows * case["vocab"]}
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    new, past = _lengths(case)
    tokens = sum(new)
    append = case["op"] == "append" or case.get("append", False)
    bytes_, flops = 0.0, 0.0
    if append:
        touched = sum((n + p - 1) // _BLOCK - p // _BLOCK + 1 for n, p in zip(new, past))
        # new keys and values, read in 16 bits and written in 8; the blocks they went to, read in 8 bits and given out in 16
        bytes_ += tokens * 2.0 * kvh * d * 3 + touched * 2.0 * kvh * (_BLOCK * d * 3 + 8)
        flops += tokens * 4.0 * kvh * d
    if case["op"] == "append":
        if case["rope"]:
            bytes_ += tokens * ((h + kvh) * 2.0 + h * 2.0) * d                # q read too, q and k written in 16 bits
            flops += tokens * 3.0 * (h + kvh) * d
        return {"bytes": bytes_, "flops": flops}
    for n, p in zip(new, past):
        ctx = n + p
        bytes_ += 2.0 * ctx * kvh * d + 8.0 * -(-ctx // _BLOCK) * kvh + n * h * d * 4.0
        flops += 4.0 * h * d * (n * p + n * (n + 1) / 2)
    return {"bytes": bytes_, "flops": flops}
