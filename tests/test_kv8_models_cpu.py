"""An 8-bit KV cache under the models and deployments that serve from it beside
plain dense ones, on CPU: q / k norms, routed experts, tensor-parallel ranks."""

import json
import os
import subprocess
import sys

import pytest
import torch

from infera_b200.engine.llm_engine import EngineConfig, LLMEngine
from infera_b200.engine.request import SamplingParams
from infera_b200.ops import kv8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
D = 128
KEYS = (5, 70, 33)
SIZES = dict(num_pages=64, max_batched_tokens=24, max_num_seqs=4)


def prompts():
    g = torch.Generator().manual_seed(3)
    return [torch.randint(2, 1024, (n,), generator=g).tolist() for n in KEYS]


def layer(eng, i):
    """fp32 (K, V) of a layer's slots."""
    k, v = eng.runner.k_cache, eng.runner.v_cache
    return (k[i].dequant(), v[i].dequant()) if isinstance(k, kv8.KV8Cache) else (k[i].float(), v[i].float())


def check_stored(x, y):
    """``x`` holds in 8 bits what ``y`` holds in bf16: an element is off by half a step of e4m3 (2^-4 of it; 2^-10 of the
    scale below the normals, and the scale is at most 2^-7 of its page's largest element; once more where a page's
    scale grew), and by a step of bf16 where products were summed in another order."""
    used = y.abs().sum(-1) > 0
    whole = sum(n // 16 * 16 for n in KEYS)  # (a finished prompt's last page, if not full, may hold another's rows)
    assert int(used.sum()) >= whole and torch.equal(used, x.abs().sum(-1) > 0)
    heads = y.shape[-1] // D
    page = y.view(-1, 16, heads, D).abs().amax(dim=(1, 3))[:, None, :, None].expand(-1, 16, heads, D).reshape(y.shape)
    assert bool(((x - y).abs() <= y.abs() * (2 ** -4 + 2 ** -7) + (2 * 2 ** -17 + 2 ** -20) * page).all())


@pytest.mark.parametrize("model,over", [("tiny-dense", {"qk_norm": True}), ("tiny-moe-gqa", {}),
                                        ("tiny-moe-gqa", {"qk_norm": True, "moe_softmax": True}), ("tiny-dense-fp8", {})])
def test_models(model, over):
    """The first layer's K and V depend on tokens and positions alone; the second's come after an attention over 8-bit
    codes, and are off by less than the largest relative rounding of a stored element, 2^-4, on top of their own (2^-4
    at most for each element)."""
    engines = [LLMEngine(EngineConfig(model=model, use_cuda_graphs=False, kv_cache_dtype=kv, model_overrides=dict(over),
                                      **SIZES), device="cpu") for kv in ("fp8", "bf16")]
    for e in engines:
        assert [len(o) for o in e.generate(prompts(), SamplingParams(max_tokens=1, ignore_eos=True))] == [1, 1, 1]
    assert isinstance(engines[0].runner.k_cache, kv8.KV8Cache)
    for x, y in zip(*[layer(e, 0) for e in engines]):
        check_stored(x, y)
    for x, y in zip(*[layer(e, 1) for e in engines]):
        assert float((x - y).norm() / y.norm()) < 2 ** -3
    # and goes on with single tokens
    longer = [p + [7, 8] for p in prompts()]
    assert [len(o) for o in engines[0].generate(longer, SamplingParams(max_tokens=6, ignore_eos=True))] == [6, 6, 6]


def test_data_parallel_engine_takes_or_refuses_it():
    from infera_b200.engine.dp_attention import DPAttentionEngine, EPSpec

    one = EPSpec(0, 1, group=None, gloo=None, fused=False)
    cfg = lambda model: EngineConfig(model=model, use_cuda_graphs=False, kv_cache_dtype="fp8", **SIZES)  # noqa: E731
    with pytest.raises(ValueError, match="fp8 KV cache"):
        DPAttentionEngine(cfg("tiny-moe"), one, device="cpu")
    assert isinstance(DPAttentionEngine(cfg("tiny-moe-gqa"), one, device="cpu").engine.runner.k_cache, kv8.KV8Cache)


def test_two_tensor_parallel_ranks():
    """Each rank stores its KV heads, as one instance with a bf16 cache stores all of them."""
    env = dict(os.environ, PYTHONPATH=ROOT)
    cmd = ["timeout", "-k", "10", "240", sys.executable, "-m", "torch.distributed.run", "--nnodes=1",
           "--nproc-per-node", "2", "--master-addr", "127.0.0.1", "--master-port", "29797", os.path.abspath(__file__)]
    r = subprocess.run(cmd, env=env, cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=300)
    out = r.stdout.decode()
    assert r.returncode == 0, out[-3000:]
    res = json.loads([x for x in out.splitlines() if x.startswith("{")][-1])
    assert res == {"ranks": 2, "outputs": [6, 6, 6]}


def rank_main():
    from datetime import timedelta

    import torch.distributed as dist

    from infera_b200.engine.tp_engine import TPLeader, follower_loop
    from infera_b200.models.config import get_config
    from infera_b200.parallel.comm import TPComm

    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    cpu = torch.device("cpu")
    dist.init_process_group("gloo", timeout=timedelta(seconds=120))
    coll, ctrl = [dist.new_group(backend="gloo", timeout=timedelta(seconds=120)) for _ in range(2)]
    tp = TPComm(rank, world, cpu, get_config("tiny-dense").hidden, nccl_group=coll, gloo_group=ctrl, max_rows=256)
    eng = LLMEngine(EngineConfig(model="tiny-dense", use_cuda_graphs=False, kv_cache_dtype="fp8", **SIZES), device=cpu,
                    tp=tp)
    lead = TPLeader(eng, ctrl) if rank == 0 else None

    def serve(n):
        if lead is None:
            follower_loop(eng, ctrl)
            return None
        outs = lead.generate(prompts(), SamplingParams(max_tokens=n, ignore_eos=True))
        lead.shutdown()
        return [len(o) for o in outs]

    serve(1)
    one = LLMEngine(EngineConfig(model="tiny-dense", use_cuda_graphs=False, **SIZES), device=cpu)
    one.generate(prompts(), SamplingParams(max_tokens=1, ignore_eos=True))
    width = eng.runner.k_cache.hkv * D if hasattr(eng.runner.k_cache, "hkv") else 0
    assert width * world == one.model_cfg.kv_size
    for x, y in zip(layer(eng, 0), layer(one, 0)):
        check_stored(x, y[:, rank * width:(rank + 1) * width])
    outs = serve(6)
    if rank == 0:
        print(json.dumps({"ranks": world, "outputs": outs}), flush=True)
    dist.barrier(group=ctrl)
    dist.destroy_process_group()


if __name__ == "__main__":
    rank_main()
