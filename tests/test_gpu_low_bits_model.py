"""A model whose feed-forwards have 4-bit weights, through the step function and the engine."""

from dataclasses import replace

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ayaka_py_b200 import GPT2Config, SamplingParams, StopCriteria
from ayaka_py_b200.microscale import matrix4


def model_of(weight_bits, dtype, rounded=False):
    """A small GPT-2 whose feed-forward matrices are 4-bit, or (``rounded``) hold the same numbers in the compute dtype."""
    from ayaka_py_b200 import models, parts  # noqa: F401
    from ayaka_py_b200.models.model import Model
    from ayaka_py_b200.parts import PartSpec
    from ayaka_py_b200.registry import architecture_for
    from ayaka_py_b200.weights.loader import DictStore, load_weights
    from ayaka_py_b200.weights.random_init import random_tensors
    config = GPT2Config(vocab_size=211, n_positions=320, n_embd=128, n_layer=2, n_head=2, n_inner=288)
    arch = architecture_for(config.to_dict())
    spec = arch.build_spec(config)
    layers = tuple(replace(layer, parts=tuple((name, PartSpec(p.kind, {**p.params, "weight_bits": weight_bits}, p.sources) if name == "ffn" else p)
                                              for name, p in layer.parts)) for layer in spec.layers)
    tensors = random_tensors(arch, config, 3, dtype="float32", device="cpu")
    for name in tensors:
        if tensors[name].ndim == 2:
            tensors[name] = tensors[name] * 4.0
        if rounded and ".mlp." in name and tensors[name].ndim == 2:
            tensors[name] = matrix4(tensors[name].T).decoded().T.contiguous()          # stored [in, out]
    if dtype == torch.bfloat16:
        tensors = {name: t.to(torch.bfloat16) for name, t in tensors.items()}
    model = Model(replace(spec, layers=layers), dtype, "cuda")
    load_weights(model, DictStore(tensors), arch.normalize_name, config)
    return model


def logits_of(model, steps):
    from ayaka_py_b200.cache.manager import CacheManager
    from ayaka_py_b200.engine.step import StepEntry, StepRunner
    cache = CacheManager(model.groups, kv_pages=64, page_size=16, max_requests=4, max_len=320, dtype=model.dtype, device="cuda")
    runner, slots, out = StepRunner(model, cache, max_tokens=640), {}, []
    for step in steps:
        entries = []
        for rid, tokens in step:
            if rid not in slots:
                slots[rid] = cache.open(rid)
            entries.append(StepEntry(slots[rid], int(cache.length[slots[rid]]), tokens, list(range(len(tokens)))))
        reservation = cache.reserve([(e.slot, e.start, len(e.tokens)) for e in entries])
        out.append(runner.run(entries).double().clone())
        cache.commit(reservation)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_of_prompts_and_single_tokens(dtype):
    """Against the same numbers in 32-bit.  A number rounded to e4m3 is off by 1 / (16 sqrt 3) of its power of two in the root mean
    square, 1 / (16 sqrt 6) = 0.0255 of itself over mantissas spread evenly.  A feed-forward rounds the rows of both its products; the
    first rounding passes the activation, whose relative slope z gelu'(z) / gelu(z) is 1 at 0 and at most 2 or so where gelu is not
    small: 0.0255 sqrt(1 + 1.6^2) = 0.048 of its output.  Two layers, and streams that are feed-forward outputs at most: 0.048 sqrt 2
    = 0.068.  In bfloat16 the usual 0.02 beside it."""
    from ayaka_py_b200 import ops
    rs = np.random.RandomState(1)
    steps = [[("a", rs.randint(0, 211, 130).tolist()), ("b", rs.randint(0, 211, 21).tolist())]]
    steps += [[("a", [int(rs.randint(211))]), ("b", [int(rs.randint(211))])] for _ in range(3)]
    steps += [[("a", [7]), ("c", rs.randint(0, 211, 70).tolist())]]
    small, large = model_of(4, dtype), model_of(16, torch.float32, rounded=True)
    matrices = 2 * 2 * 128 * 288                              # numbers of the feed-forwards' weights, 4 bytes each in the one model
    assert small.weight_bytes() < large.weight_bytes() - 4 * matrices + matrices
    got, want = logits_of(small, steps), logits_of(large, steps)
    assert ops.tc_error() == 0
    for g, w in zip(got, want):
        assert float((g - w).norm() / w.norm()) < (0.07 if dtype == torch.float32 else 0.09)


@pytest.mark.parametrize("decode_graph", [True, False])
def test_generation(decode_graph):
    """The engine's steps (captured and replayed, or one by one) give the tokens of a replay of the same steps."""
    from ayaka_py_b200.config.engine import EngineConfig
    from ayaka_py_b200.engine.engine import Engine
    from ayaka_py_b200.engine.request import Request
    model = model_of(4, torch.float32)
    engine = Engine(model, EngineConfig(dtype="float32", kv_pages=64, batch_tokens=64, prefill_chunk=32, decode_graph=decode_graph))
    prompts = [list(range(3, 40)), [9, 8, 7]]
    for i, p in enumerate(prompts):
        engine.submit(Request(f"r{i}", p, SamplingParams(temperature=0.0), StopCriteria(max_tokens=12, ignore_eos=True)))
    done = engine.run_until_idle()
    for i, p in enumerate(prompts):
        tokens = done[f"r{i}"].token_ids
        logits = logits_of(model, [[("x", p + tokens)]])[0][len(p) - 1:-1]
        slack = 2.0 ** -10 * float(logits.abs().max())            # sums of another order, rounded to 8 bits here and there to the neighbour
        best = logits.max(-1).values
        taken = logits[torch.arange(len(tokens)), torch.tensor(tokens)]
        assert len(tokens) == 12 and bool((taken >= best - 16 * slack).all())
    engine.cache.assert_clean()
