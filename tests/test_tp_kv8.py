"""The 8-bit KV cache and log probabilities on tensor-parallel ranks (gloo, CPU)."""
import json

import pytest

from test_tp_cpu import launch


@pytest.mark.parametrize("world,precision,port", [(2, "int8", 29631), (4, "fp8", 29632)])
def test_ranks_with_an_8_bit_cache_answer_like_one(tmp_path, world, precision, port):
    """Each rank keeps its own heads' codes, whose scales no other head shares, so that the shards hold what one rank would;
    the vocabulary's shards are gathered for the figures, which every rank reports alike."""
    out = tmp_path / "r.json"
    p = launch(world, "kv8_engine_worker.py", [precision, str(out)], port)
    assert p.returncode == 0, p.stderr[-3000:]
    r = json.loads(out.read_text())
    assert r["same"] and r["heads"] == 4 // world
    for (toks, lps), (want, lps1) in zip(r["tp"], r["single"]):
        assert toks == want and (lps is None) == (lps1 is None)
        for (t, lp, rank, ent, top), (t1, lp1, rank1, ent1, top1) in zip(lps or [], lps1 or []):
            # fp32 sums in another order
            assert t == t1 and rank == rank1 == 1 and abs(lp - lp1) < 1e-4 and abs(ent - ent1) < 1e-4
            assert [i for i, _ in top] == [i for i, _ in top1] and all(i < 999 for i, _ in top)
    assert [len(lps or []) for _, lps in r["tp"]] == [20, 20, 0, 20] and [len(lps[0][4]) for _, lps in r["tp"] if lps] == [3, 0, 5]
    for toks, lps in r["drawn"]:
        assert all(t == x[0] and x[1] <= 0 and x[2] >= 1 for t, x in zip(toks, lps or []))
