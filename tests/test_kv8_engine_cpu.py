"""The engine over an 8-bit KV cache, on CPU: what its steps store, its
answers next to a bf16 cache's, and the configurations that it refuses."""

import pytest
import torch

from infera_b200.engine.llm_engine import EngineConfig, LLMEngine
from infera_b200.engine.request import SamplingParams
from infera_b200.ops import kv8


def engine(kv="fp8", **kw):
    cfg = EngineConfig(model=kw.pop("model", "tiny-dense"), use_cuda_graphs=False, kv_cache_dtype=kv, **kw)
    return LLMEngine(cfg, device="cpu")


def prompts(*lens):
    g = torch.Generator().manual_seed(3)
    return [torch.randint(2, 1024, (n,), generator=g).tolist() for n in lens]


def first_layer(eng):
    """fp32 (K, V) of the first layer's slots."""
    k, v = eng.runner.k_cache, eng.runner.v_cache
    return (k[0].dequant(), v[0].dequant()) if isinstance(k, kv8.KV8Cache) else (k[0].float(), v[0].float())


def test_cache_holds_what_a_bf16_cache_holds():
    """The first layer's K and V depend on tokens and positions alone, so both engines put the same values into the same
    slots: an element is off by half a step of e4m3 (2^-4 of it; 2^-10 of the scale below the normals, and the scale is
    at most 2^-7 of its page's largest element; once more where a page's scale grew) and half a step of bf16."""
    ask = prompts(5, 70, 33)
    a, b = [engine(kv, num_pages=64, max_batched_tokens=24, max_num_seqs=4) for kv in ("fp8", "bf16")]
    # the same tokens on both sides, whatever the engines would choose
    outs = [e.generate(ask, SamplingParams(max_tokens=1, ignore_eos=True)) for e in (a, b)]
    assert [len(o) for o in outs[0]] == [1, 1, 1]
    for x, y in zip(first_layer(a), first_layer(b)):
        used = y.abs().sum(-1) > 0
        assert int(used.sum()) >= 96 and torch.equal(used, x.abs().sum(-1) > 0)
        page = y.view(-1, 16, 2, 128).abs().amax(dim=(1, 3))[:, None, :, None].expand(-1, 16, 2, 128).reshape(y.shape)
        assert bool(((x - y).abs() <= y.abs() * (2 ** -4 + 2 ** -8) + 2 * 2 ** -10 * 2 ** -7 * page).all())


def test_answers_stand_next_to_a_bf16_cache():
    """Logits after a prompt in chunks: off by less than the largest relative rounding of a stored element, 2^-4."""
    ask = prompts(60)
    logits = []
    for kv in ("fp8", "bf16"):
        e = engine(kv, num_pages=64, max_batched_tokens=24, max_num_seqs=4)
        e.generate(ask, SamplingParams(max_tokens=1, ignore_eos=True))
        logits.append(e.runner.last_logits.float())
    x, y = logits
    assert float((x - y).norm() / y.norm()) < 2 ** -4


def test_prefix_pages_are_shared_and_recycled():
    """Cached pages serve a second request; a pool too small for all keeps recycling pages, whose old scales are dropped
    when their first slot is written."""
    eng = engine(num_pages=12, max_batched_tokens=256, max_num_seqs=2)
    long = prompts(64)[0]
    sp = SamplingParams(max_tokens=4, ignore_eos=True)
    first = eng.generate([long + [1, 2, 3]], sp)[0]
    before = eng.bm.stats["hit_tokens"]
    again = eng.generate([long + [1, 2, 3]], sp)[0]
    assert eng.bm.stats["hit_tokens"] - before >= 48 and again == first
    for p in prompts(90, 100, 80, 70):
        assert len(eng.generate([p], sp)[0]) == 4
    fresh = engine(num_pages=12, max_batched_tokens=256, max_num_seqs=2)
    assert eng.generate([long + [7]], sp) == fresh.generate([long + [7]], sp)


@pytest.mark.parametrize("kw", [dict(kv="int8"), dict(kv_tier="pinned:1"), dict(disagg_mode="decode"),
                                dict(disagg_mode="prefill"), dict(page_size=32), dict(model="tiny-moe"),
                                dict(model_overrides={"head_dim": 64}), dict(model_overrides={"num_heads": 18})])
def test_refusals(kw):
    with pytest.raises(ValueError):
        engine(**kw)


def test_launcher_passes_the_choice_on():
    from infera_b200.engine import worker

    args = worker.parse_args(["--model", "tiny-dense", "--kv-cache-dtype", "fp8"])
    cmd = worker._core_cmd(args, "ipc://a", "ipc://b")
    assert cmd[cmd.index("--kv-cache-dtype") + 1] == "fp8"
