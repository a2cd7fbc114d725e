"""MXFP4 off the GPU: the CPU definition's known answers, and calls that are refused before
anything reaches a kernel."""

import ctypes

import pytest
import torch

from oracle import mxfp4
from tokserve_amd.engine.paged.storage import PagedKVStorage
from tokserve_amd.kernels import _lib, ops, torch_ops

CODES, SCALES = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def test_known_codes() -> None:
    """Borders between codes, ties to the even code, saturation, the scale's rule."""

    x = torch.zeros(5, 32)
    x[0, :9] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.26])
    x[1, :3] = torch.tensor([7.9, -7.9, 4.9])
    x[2, 0] = 1e-45
    x[3, 4] = float("inf")
    x[4, 1] = 2.0 ** 127
    codes, scales = mxfp4.quantize(x)
    assert scales[:, 0].tolist() == [127, 127, 2, 255, 252]
    back = mxfp4.values(codes, scales)
    assert back[0, :9].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.5]
    assert back[1, :3].tolist() == [6.0, -6.0, 4.0]
    assert not back[2].any() and torch.isnan(back[3]).all() and back[4, 1] == 2.0 ** 127
    assert codes[0, 0] == 6 and codes[0, 4] == 9  # element 0 in the low nibble; -0.5


def test_every_operator_is_registered_with_its_writes_marked() -> None:
    writes = {"mxfp4_quantize": {"codes", "scales"}, "mxfp4_dequantize": {"out"},
              "mxfp4_matmul": {"out", "workspace"}, "mxfp4_linear": {"out", "workspace"}}
    assert set(torch_ops.MXFP4_SCHEMAS) == set(writes)
    for name, expected in writes.items():
        schema = getattr(torch.ops.tokserve_amd, name).default._schema
        assert {a.name for a in schema.arguments
                if a.alias_info is not None and a.alias_info.is_write} == expected
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"tokserve_amd::{name}", "CUDA")


def test_cpu_tensors_are_refused() -> None:
    codes, scales = torch.empty(4, 16, dtype=CODES), torch.empty(4, 1, dtype=SCALES)
    for call in (lambda: ops.mxfp4_quantize(torch.zeros(4, 32)),
                 lambda: ops.mxfp4_dequantize(codes, scales, torch.float32),
                 lambda: ops.mxfp4_matmul(codes, scales, codes, scales, torch.float32),
                 lambda: ops.mxfp4_linear(torch.zeros(4, 32), codes, scales)):
        with pytest.raises(ValueError, match="requires HIP device tensors"):
            call()


@pytest.fixture
def fake():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        yield lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="cuda")


def test_matrices_that_are_refused(fake) -> None:
    codes, scales = fake(4, 32, dtype=CODES), fake(4, 2, dtype=SCALES)
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.mxfp4_quantize(fake(4, 48))
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        ops.mxfp4_quantize(fake(4, 64, dtype=torch.int32))
    with pytest.raises(TypeError, match="float4_e2m1fn_x2"):
        ops.mxfp4_dequantize(fake(4, 32, dtype=torch.uint8), scales, torch.float32)
    with pytest.raises(TypeError, match="out must be float32"):
        ops.mxfp4_dequantize(codes, scales, torch.float64)
    with pytest.raises(ValueError, match="one entry per 32"):
        ops.mxfp4_dequantize(codes, fake(4, 1, dtype=SCALES), torch.float32)
    with pytest.raises(ValueError, match="contiguous"):
        ops.mxfp4_dequantize(fake(8, 32, dtype=CODES)[::2], scales, torch.float32)
    with pytest.raises(ValueError, match="the inputs' K"):
        ops.mxfp4_linear(fake(3, 32), codes, scales)
    with pytest.raises(ValueError, match="have A's K"):
        ops.mxfp4_matmul(codes, scales, fake(4, 16, dtype=CODES), fake(4, 1, dtype=SCALES),
                         torch.float32)
    with pytest.raises(ValueError, match="at least one row"):
        ops.mxfp4_linear(fake(3, 64), fake(0, 32, dtype=CODES), fake(0, 2, dtype=SCALES))
    with pytest.raises(ValueError, match="out must have shape"):
        ops.mxfp4_linear(fake(3, 64), codes, scales, out=fake(3, 5))
    with pytest.raises(ValueError, match="the inputs' dtype"):
        ops.mxfp4_linear(fake(3, 64), codes, scales, out=fake(3, 4, dtype=torch.float16))
    with pytest.raises(ValueError, match="the given dtype"):
        ops.mxfp4_dequantize(codes, scales, torch.float16, out=fake(4, 64))
    with pytest.raises(ValueError, match="go together"):
        ops.mxfp4_quantize(fake(4, 64), codes=codes)
    with pytest.raises(ValueError, match="shape \\(..., K / 2\\)"):
        ops.mxfp4_quantize(fake(3, 64), codes=codes, scales=scales)
    with pytest.raises(ValueError, match="must be contiguous"):
        ops.mxfp4_linear(fake(3, 2, 64), codes, scales, out=fake(3, 2, 8)[..., :4])
    with pytest.raises(ValueError, match="workspace must be"):
        ops.mxfp4_linear(fake(3, 64), codes, scales, workspace=fake(100))
    assert ops.mxfp4_linear(fake(3, 2, 64), codes, scales).shape == (3, 2, 4)


def test_pools_that_are_refused(fake) -> None:
    def pools(dh=64, dtype=CODES):
        return fake(1, 4, 2, 16, dh // 2, dtype=dtype), fake(1, 4, 2, 16, dh // 2, dtype=dtype)

    rows, slots = fake(3, 2, 64), fake(3, dtype=torch.int64)
    scales = {n: fake(1, 4, 2, 16, 2, dtype=SCALES) for n in ("k_scales", "v_scales")}
    ops.kv_append(rows, rows, *pools(), slots, 0, **scales)
    with pytest.raises(ValueError, match="need k_scales and v_scales"):
        ops.kv_append(rows, rows, *pools(), slots, 0)
    with pytest.raises(ValueError, match="go together"):
        ops.kv_append(rows, rows, *pools(), slots, 0, k_scales=scales["k_scales"])
    with pytest.raises(TypeError, match="float8_e8m0fnu"):
        ops.kv_append(rows, rows, *pools(), slots, 0, k_scales=scales["k_scales"],
                      v_scales=fake(1, 4, 2, 16, 2))
    with pytest.raises(ValueError, match="Dh / 32"):
        ops.kv_append(rows, rows, *pools(), slots, 0, k_scales=scales["k_scales"],
                      v_scales=fake(1, 4, 2, 16, dtype=SCALES))
    with pytest.raises(ValueError, match="head_dim of 32"):
        ops.kv_append(fake(3, 2, 48), fake(3, 2, 48), *pools(48), slots, 0, **scales)
    with pytest.raises(ValueError, match="fp8 KV pools only"):
        ops.kv_append(rows, rows, *pools(), slots, 0, k_scale=2.0, **scales)
    with pytest.raises(ValueError, match="must match the pool's"):
        ops.kv_append(fake(3, 2, 32), fake(3, 2, 32), *pools(), slots, 0, **scales)
    query, tables, lens = fake(2, 4, 64), fake(2, 3, dtype=torch.int32), fake(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="same dtype"):
        ops.paged_attention_decode_noalloc(query, *pools(), tables, lens, layer_index=0,
                                           max_seq_len=40, out=fake(2, 4, 64))


def test_storage_of_mxfp4_pools() -> None:
    def storage(**more):
        return PagedKVStorage(**{**dict(num_layers=2, num_blocks=3, num_key_value_heads=2,
                                        block_size=4, head_dim=64, device=torch.device("cpu"),
                                        dtype=torch.bfloat16, kv_dtype=CODES), **more})

    pool = storage()
    assert pool.key_storage.shape == (2, 3, 2, 4, 32) and pool.key_storage.dtype == CODES
    assert pool.scales["v_scales"].shape == (2, 3, 2, 4, 2)
    assert pool.head_dim == 64 and pool.key_scales.dtype == SCALES
    with pytest.raises(ValueError, match="head_dim of 32"):
        storage(head_dim=80)
    with pytest.raises(ValueError, match="fp8 pools only"):
        storage(k_scale=2.0)
    with pytest.raises(ValueError, match="per-row scales need fp8"):
        storage(scale_granularity="row")


def test_c_entries_check_before_any_launch() -> None:
    library = _lib.load()
    here = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(here) + 15) & ~15
    value, kind, index, space = (_lib.TKS_ERR_VALUE, _lib.TKS_ERR_TYPE, _lib.TKS_ERR_INDEX,
                                 _lib.TKS_ERR_WORKSPACE)
    quantize = library.tks_mxfp4_quantize
    assert quantize(p, 32, 1, 32, p, p, 3, None) == kind
    assert quantize(p, 32, 1, 33, p, p, 0, None) == value
    assert quantize(None, 32, 1, 32, p, p, 0, None) == value
    assert quantize(p, 32, 1, 32, p + 2, p, 0, None) == value
    assert quantize(p, 32, 1 << 60, 32, p, p, 0, None) == value
    assert quantize(None, 32, 0, 32, None, None, 0, None) == _lib.TKS_OK
    assert library.tks_mxfp4_dequantize(p, p, 1, 0, p, 32, 0, None) == value
    assert library.tks_mxfp4_matmul_workspace_bytes(1, 1, 31) == -1
    assert library.tks_mxfp4_matmul(p, p, p, p, 1, 1, 48, p, 1, None, 0, 0, None) == value
    assert library.tks_mxfp4_matmul(p + 8, p, p, p, 1, 1, 32, p, 1, None, 0, 0, None) == value
    assert library.tks_mxfp4_matmul(p, p, p, p, 1, 1, 32, p, 1, None, 0, 5, None) == kind
    assert library.tks_mxfp4_linear(p, 32, p, p, 1, 1, 32, p, 1, None, 0, 0, None) == space
    append = library.tks_kv_append_mxfp4
    pool = lambda **k: [p, 64, 64, p, 64, 64, k.get("n", 1), p, p, p, p, 1, 1, 1, 16,  # noqa: E731
                        k.get("dh", 64), k.get("layer", 0), p, k.get("dtype", 0), None]
    assert append(*pool(dh=48)) == value and append(*pool(dh=160)) == value
    assert append(*pool(layer=1)) == index and append(*pool(dtype=9)) == kind
    assert append(*pool(n=0)) == _lib.TKS_OK and append(*pool(n=-1)) == value
    decode = library.tks_paged_attention_decode_mxfp4
    args = lambda **k: [p, 64, 64, p, p, p, p, 1, 4, 1, 16, 64, 0, p, k.get("width", 4), p,  # noqa: E731
                        None, 1, k.get("heads", 4), k.get("keys", 64), 1.0, k.get("pages", 0), p,
                        64, 64, None, 0, 0, None]
    assert decode(*args(keys=65)) == value and decode(*args(heads=17)) == value
    assert decode(*args(pages=1)) == space
    # A layer of 2^31 rows or more: blocks of 16 tokens only.
    many = args(width=64)
    many[8], many[10] = 1 << 31, 1
    assert decode(*many) == value
    prefill = library.tks_paged_attention_prefill_mxfp4_workspace_bytes
    assert prefill(2, 4, 4, 1, 64, 16, 40, 0) == 0  # (fp32: straight from the pools)
    assert prefill(2, 511, 4, 1, 128, 16, 512, 2) == 0 == prefill(2, 512, 4, 1, 128, 16, 511, 2)
    assert prefill(2, 512, 4, 1, 128, 16, 512, 2) == \
        2 * (2 * 32 * 16 * 128 * 2) + 256 + 1024  # K, V, the table, a byte per row
    assert prefill(2, 512, 4, 1, 96, 16, 512, 2) == 0 == prefill(2, 512, 4, 1, 128, 24, 512, 2)
    assert prefill(2, 512, 4, 1, 64, 16, 512, 2) == 0 < prefill(2, 2048, 4, 1, 64, 16, 1024, 2)
    assert prefill(64, 1 << 20, 8, 8, 128, 16, 1 << 15, 2) == 0  # (too much of it)
    assert prefill(2, 512, 4, 3, 128, 16, 512, 2) == -1


def test_projections_on_the_cpu() -> None:
    from tokserve_amd.engine.config import LlamaConfig
    from tokserve_amd.engine.layers import MXFP4Linear
    from tokserve_amd.engine.model import LlamaModel

    module = MXFP4Linear(64, 10)
    assert module.codes.shape == (10, 32) and module.scales.shape == (10, 2)
    assert module.bfloat16().codes.dtype == torch.uint8
    assert list(module.state_dict()) == ["codes", "scales"]
    with pytest.raises(ValueError, match="multiple of 32"):
        MXFP4Linear(48, 10)
    with pytest.raises(ValueError, match="out_features"):
        MXFP4Linear(32, 0)
    with pytest.raises(ValueError, match="requires HIP device"):
        module(torch.zeros(1, 64))
    sizes = dict(vocab_size=50, num_hidden_layers=1, num_attention_heads=2,
                 num_key_value_heads=1, max_position_embeddings=64)
    with pytest.raises(ValueError, match="hidden_size to be a multiple of 32"):
        LlamaModel(LlamaConfig(hidden_size=40, intermediate_size=64, **sizes)).quantize_mxfp4()
    model = LlamaModel(LlamaConfig(hidden_size=64, intermediate_size=96, **sizes))
    with pytest.raises(ValueError, match="requires HIP device"):
        model.quantize_mxfp4()
    assert model.weights_version == 0
    assert isinstance(model.layers[0].mlp.up_proj, torch.nn.Linear)
