"""Child process of the tensor-parallel tests: the serving engine with an 8-bit KV cache and log probabilities at the launched
world size, beside one rank with the same seeded model."""
import json
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))

import torch  # noqa: E402

from ronn_b200.api.model import Model  # noqa: E402
from ronn_b200.models.gpt2 import GPT2Config, build_gpt2  # noqa: E402
from ronn_b200.parallel import make_comm  # noqa: E402
from ronn_b200.parallel.group import init_distributed  # noqa: E402
from ronn_b200.serving import EngineConfig, LLMEngine, SamplingParams  # noqa: E402


def main():
    precision, out_path = sys.argv[1:3]
    rank, world, _ = init_distributed("gloo", timeout_s=120)
    # 999 tokens: the last rank's shard of the vocabulary is padded
    model = Model.from_graph(build_gpt2(GPT2Config.tiny(n_layer=2, n_embd=256, n_head=4, vocab_size=999, n_positions=256),
                                        dtype=torch.float32, seed=7))
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 999, (n,), generator=g).tolist() for n in (5, 17, 40, 33)]

    def run(comm, **how):
        eng = LLMEngine(model, EngineConfig(max_num_seqs=8, max_batch_tokens=64, max_model_len=256, dtype="fp32", backend="torch",
                                            kv_cache_dtype=precision, tp_size=world if comm else 1, tp_comm="nccl", num_blocks=64,
                                            use_cuda_graph=False), device=torch.device("cpu"), comm=comm)
        ids = [eng.add_request(p, SamplingParams(max_new_tokens=20, logprobs=n, **how)) for p, n in zip(prompts, (3, 0, None, 5))]
        while eng.has_unfinished():
            eng.step()
        heads = eng.runner.kcache[0].shape[1]
        return heads, [(eng.requests[i].output_tokens, None if eng.requests[i].output_logprobs is None else
                        [(p.token, p.logprob, p.rank, p.entropy, p.top) for p in eng.requests[i].output_logprobs]) for i in ids]

    comm = make_comm("nccl", torch.device("cpu"))
    heads, tp = run(comm)
    _, single = run(None)
    _, drawn = run(comm, temperature=0.8, top_k=50, repeat_penalty=1.2, seed=11)
    gathered = [None] * world
    torch.distributed.all_gather_object(gathered, (tp, drawn))
    if rank == 0:
        with open(out_path, "w") as f:
            json.dump({"tp": tp, "single": single, "drawn": drawn, "heads": heads, "same": all(x == gathered[0] for x in gathered)}, f)
    torch.distributed.barrier()
    torch.distributed.destroy_process_group()


if __name__ == "__main__":
    main()
