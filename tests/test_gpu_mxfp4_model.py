"""MXFP4 weights and K/V pools in the model and the engine.

Every product of a run is checked against 64-bit sums of the decoded values (its inputs
rounded by the CPU definition) with the bound that test_gpu_mxfp4.py derives: K / 128 + 15
steps of 2^-23 of sum |a b|, and half a step of the result's type.
"""

import copy

import pytest
import torch

from oracle import mxfp4
from tokserve_amd.batching.engine import ContinuousBatchEngine
from tokserve_amd.engine.config import LlamaConfig
from tokserve_amd.engine.layers import MXFP4Linear, SwiGLU
from tokserve_amd.engine.model import LlamaModel
from tokserve_amd.engine.paged.manager import PagedKVCacheManager
from tokserve_amd.generation.paged_generate import generate_with_paged_cache
from tokserve_amd.generation.types import GenerationConfig
from tokserve_amd.kernels import ops
from tokserve_amd.scheduler.request import ScheduledRequest
from tokserve_amd.scheduler.scheduler import RequestScheduler

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CONFIG = LlamaConfig(vocab_size=97, hidden_size=256, intermediate_size=416, num_hidden_layers=2,
                     num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=128)
SPECS = (("A", [1, 2, 3], 9), ("B", list(range(4, 44)), 6), ("C", [8], 12), ("D", [9] * 17, 5))


def _model(device, dtype) -> LlamaModel:
    torch.manual_seed(7)
    return LlamaModel(CONFIG).to(device=device, dtype=dtype).eval()


def _manager(device, dtype, kv_dtype=torch.float4_e2m1fn_x2) -> PagedKVCacheManager:
    return PagedKVCacheManager(num_layers=CONFIG.num_hidden_layers, num_blocks=24,
                               num_key_value_heads=CONFIG.num_key_value_heads, block_size=16,
                               head_dim=CONFIG.head_dim, device=device, dtype=dtype,
                               kv_dtype=kv_dtype)


def _engine(model, device, *, overlap=False, graphs=True):
    """graphs=False: the same launches, none of them captured."""

    manager = _manager(device, model.embed_tokens.weight.dtype)
    scheduler = RequestScheduler(max_running_requests=3, cache_manager=manager)
    engine = ContinuousBatchEngine(model, scheduler, manager, overlap_decode=overlap)
    if not graphs:
        engine.executor.graphs.max_graphs = 0
    return engine


def _run(engine, device, run=0) -> list[list[int]]:
    for rid, prompt, n in SPECS:
        engine.scheduler.submit(ScheduledRequest(f"{rid}{run}",
                                                 torch.tensor([prompt], device=device),
                                                 GenerationConfig(max_new_tokens=n)))
    engine.run_until_idle()
    return [r.token_ids.flatten().tolist() for r in engine.results[-len(SPECS):]]


def _check_products(calls) -> None:
    for inputs, codes, scales, out in calls:
        a = mxfp4.values(*mxfp4.quantize(inputs.cpu().reshape(-1, inputs.shape[-1])))
        b = mxfp4.values(codes.cpu(), scales.cpu())
        exact, size = a @ b.t(), a.abs() @ b.abs().t()
        limit = ((a.shape[1] / 128 + 15) * 2.0 ** -23 * size
                 + torch.finfo(out.dtype).eps / 2 * exact.abs() + torch.finfo(out.dtype).tiny)
        assert bool(((out.cpu().double().view_as(exact) - exact).abs() <= limit).all())


@pytest.fixture
def products(monkeypatch):
    """Copies of every product's inputs and result."""

    calls = []
    linear = ops.mxfp4_linear

    def recorded(inputs, codes, scales, **kw):
        out = linear(inputs, codes, scales, **kw)
        calls.append(tuple(t.clone() for t in (inputs, codes.view(torch.uint8),
                                               scales.view(torch.uint8), out)))
        return out

    monkeypatch.setattr(ops, "mxfp4_linear", recorded)
    return calls


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_projection(device, dtype, products) -> None:
    torch.manual_seed(1)
    linear = torch.nn.Linear(96, 40, bias=False, device=device, dtype=dtype)
    module = MXFP4Linear.from_linear(linear)
    codes, scales = mxfp4.quantize(linear.weight)
    assert torch.equal(module.codes.cpu(), codes) and torch.equal(module.scales.cpu(), scales)
    x = torch.randn(2, 3, 96, device=device, dtype=dtype)
    out = module(x)
    assert out.shape == (2, 3, 40) and out.dtype == dtype
    _check_products(products)
    # Bytes stay bytes under a change of type, and a state dict carries them.
    other = MXFP4Linear(96, 40).to(device=device, dtype=torch.float16)
    other.load_state_dict(module.half().state_dict())
    assert torch.equal(other(x), out)
    with pytest.raises(ValueError, match="bias"):
        MXFP4Linear.from_linear(torch.nn.Linear(32, 8, device=device))


@pytest.mark.parametrize("tokens", [1, 5, 70])
def test_feed_forward_is_its_parts(device, tokens, products) -> None:
    """Gate and up as one product over stacked rows, which the two modules still own."""

    torch.manual_seed(2)
    mlp = SwiGLU(64, 160).to(device=device, dtype=torch.bfloat16)
    for name, linear in list(mlp.named_children()):
        setattr(mlp, name, MXFP4Linear.from_linear(linear))
    before = copy.deepcopy(mlp.state_dict())
    x = torch.randn(tokens, 64, device=device, dtype=torch.bfloat16)
    with torch.inference_mode():
        out = mlp(x)
        assert torch.equal(mlp(x), out)
    _check_products(products)
    (first, _, _, gate_up), (hidden, _, _, last) = products[:2]
    assert torch.equal(first, x) and gate_up.shape == (tokens, 320) and torch.equal(last, out)
    assert torch.equal(hidden, ops.silu_mul(gate_up))
    after = mlp.state_dict()
    assert all(torch.equal(after[name], before[name]) for name in before)
    assert mlp.up_proj.codes.data_ptr() == mlp.gate_proj.codes.data_ptr() + mlp.gate_proj.codes.numel()
    # New weights come in through the modules' buffers; a moved module is stacked anew.
    mlp.load_state_dict({name: t.flip(0) for name, t in before.items()})
    with torch.inference_mode():
        turned = mlp(x)
        assert torch.equal(copy.deepcopy(mlp)(x), turned)
    assert not torch.equal(turned, out)
    _check_products(products)


@pytest.mark.parametrize("dtype", DTYPES)
def test_engine_over_mxfp4_weights_and_pools(device, dtype, products) -> None:
    """A whole run, its products against the CPU; replayed from graphs and overlapped it gives
    the same tokens."""

    model = _model(device, dtype).quantize_mxfp4()
    engine = _engine(model, device, graphs=False)
    expected = _run(engine, device)
    assert sorted(map(len, expected)) == sorted(len(prompt) + n for _, prompt, n in SPECS)
    assert len(products) == 4 * CONFIG.num_hidden_layers * len(engine.history)
    _check_products(products)
    assert not engine.executor.graphs._graphs
    for overlap in (False, True):
        engine = _engine(model, device, overlap=overlap)
        for run in range(2):
            assert _run(engine, device, run) == expected
            assert engine.executor.graphs._graphs


def test_one_sequence_through_the_modules(device, products) -> None:
    """The one-sequence interface: prefill, then a token at a time, each projection by itself."""

    model = _model(device, torch.float32).quantize_mxfp4()
    prompt = torch.tensor([list(range(3, 40))], device=device)
    config = GenerationConfig(max_new_tokens=6)
    manager = _manager(device, torch.float32)
    result = generate_with_paged_cache(model, prompt, config, manager, sequence_id="s")
    assert result.token_ids.shape == (1, 43)
    assert len(products) % (7 * CONFIG.num_hidden_layers - 2) == 0  # gate and up are one
    _check_products(products)
    again = generate_with_paged_cache(model, prompt, config, manager, sequence_id="t")
    assert torch.equal(again.token_ids, result.token_ids)
    assert manager.allocator.allocated_count == 0


def test_quantizing_under_captured_graphs(device) -> None:
    """Graphs of the weights from before are not replayed."""

    model = _model(device, torch.bfloat16)
    quantized = copy.deepcopy(model).quantize_mxfp4()
    expected = _run(_engine(quantized, device), device)
    engine = _engine(model, device)
    _run(engine, device)
    old = list(engine.executor.graphs._graphs.values())
    assert old
    assert model.quantize_mxfp4() is model
    state = model.state_dict()
    assert all(torch.equal(state[k], v) for k, v in quantized.state_dict().items())
    codes = model.layers[0].mlp.down_proj.codes.data_ptr()
    assert model.quantize_mxfp4().layers[0].mlp.down_proj.codes.data_ptr() == codes
    assert _run(engine, device, 1) == expected
    new = list(engine.executor.graphs._graphs.values())
    assert new and not any(graph in old for graph in new)


def test_refusals(device) -> None:
    torch.manual_seed(0)
    odd = LlamaConfig(vocab_size=50, hidden_size=64, intermediate_size=100, num_hidden_layers=1,
                      num_attention_heads=2, num_key_value_heads=1, max_position_embeddings=64)
    model = LlamaModel(odd).to(device)
    with pytest.raises(ValueError, match="intermediate_size"):
        model.quantize_mxfp4()
    assert isinstance(model.layers[0].self_attention.q_proj, torch.nn.Linear)
    double = _model(device, torch.float64)
    with pytest.raises(TypeError):
        double.quantize_mxfp4()
    assert isinstance(double.layers[0].self_attention.q_proj, torch.nn.Linear)
