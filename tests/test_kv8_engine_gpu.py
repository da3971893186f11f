"""The engine over an 8-bit KV cache on a GPU: prompts in chunks, mixed steps,
graphed and eager decode steps."""

import pytest
import torch

from infera_b200.engine.llm_engine import EngineConfig, LLMEngine
from infera_b200.engine.request import SamplingParams
from infera_b200.ops import kernels as K
from infera_b200.ops import kv8

pytestmark = pytest.mark.gpu


def engine(kv="fp8", model="tiny-dense-gpu", **kw):
    return LLMEngine(EngineConfig(model=model, kv_cache_dtype=kv, **kw), device="cuda:0")


def prompts(*lens):
    g = torch.Generator().manual_seed(3)
    return [torch.randint(2, 4096, (n,), generator=g).tolist() for n in lens]


def check_status():
    torch.cuda.synchronize()
    assert K.scratch().read_status() == 0


@pytest.mark.parametrize("model", ["tiny-dense-gpu", "tiny-dense-fp8-gpu"])
def test_cache_holds_what_a_bf16_cache_holds(model):
    """The first layer's K and V depend on tokens and positions alone. An element is off by half a step of e4m3 (2^-4 of
    it; 2^-10 of the scale below the normals, and the scale is at most 2^-7 of its page's largest element; once more
    where a page's scale grew), and by a step of bf16 where the two engines' products round differently."""
    got = []
    for kv in ("fp8", "bf16"):
        e = engine(kv, model, num_pages=64, max_batched_tokens=96, max_num_seqs=4, use_cuda_graphs=False)
        e.generate(prompts(40, 300, 33), SamplingParams(max_tokens=1, ignore_eos=True))
        check_status()
        k, v = e.runner.k_cache, e.runner.v_cache
        got.append((k[0].dequant(), v[0].dequant()) if kv == "fp8" else (k[0].float(), v[0].float()))
    for x, y in zip(*got):
        used = y.abs().sum(-1) > 0
        assert int(used.sum()) >= 320 and torch.equal(used, x.abs().sum(-1) > 0)
        page = y.view(-1, 16, 2, 128).abs().amax(dim=(1, 3))[:, None, :, None].expand(-1, 16, 2, 128).reshape(y.shape)
        assert bool(((x - y).abs() <= y.abs() * (2 ** -4 + 2 ** -7) + (2 * 2 ** -10 * 2 ** -7 + 2 ** -20) * page).all())


@pytest.mark.parametrize("graphs", [False, True])
def test_serves(graphs):
    """Prompts longer than a step, sequences that decode while others are prefilled, shared prefixes, sampled and
    padded graph batches; the next token's logits stand next to a bf16 cache's (off by less than the largest relative
    rounding of a stored element, 2^-4)."""
    eng = engine(num_pages=200, max_num_seqs=8, max_batched_tokens=96, use_cuda_graphs=graphs)
    assert isinstance(eng.runner.k_cache, kv8.KV8Cache)
    prefix = prompts(64)[0]
    ask = prompts(3, 130, 47) + [prefix + [1, 2, 3], prefix + [9, 8]]
    outs = eng.generate(ask, SamplingParams(max_tokens=20, ignore_eos=True))
    check_status()
    assert [len(o) for o in outs] == [20] * 5
    before = eng.bm.stats["hit_tokens"]
    longer = ask[1] + outs[1]
    last = eng.generate([longer], SamplingParams(max_tokens=1, ignore_eos=True))
    assert eng.bm.stats["hit_tokens"] - before >= 128 and len(last[0]) == 1
    check_status()
    x = eng.runner.last_logits.float().clone()
    ref = engine("bf16", num_pages=200, max_num_seqs=8, max_batched_tokens=256, use_cuda_graphs=False)
    ref.generate([longer], SamplingParams(max_tokens=1, ignore_eos=True))
    y = ref.runner.last_logits.float()
    assert float((x - y).norm() / y.norm()) < 2 ** -4


def test_holds_twice_the_tokens():
    """A page takes half the memory (and 1 / 2048 more for its scales)."""
    a = engine(num_pages=64, max_num_seqs=2, use_cuda_graphs=False)
    b = engine("bf16", num_pages=64, max_num_seqs=2, use_cuda_graphs=False)
    mine, bf16 = a.runner.k_cache.nbytes, b.runner.k_cache.numel() * 2
    assert bf16 / 2 < mine <= bf16 / 2 * (1 + 2 ** -11)
    assert a._derive_num_pages() > 1.9 * b._derive_num_pages()
