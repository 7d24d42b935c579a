"""Without a GPU: refusals, meta kernels and C argument checks of the attention and norm
operators, and their 64-bit definitions against torch's own on plain cases."""

import pytest
import torch

import ayaka.kernel.hip as H
from ayaka.kernel.hip import _lib
from ayaka.utils.import_utils import CapabilityError
from oracle import serving_oracle as ora

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _decode_args(**change):
    args = {"query": torch.zeros(2, 4, 64, dtype=BF16), "key_cache": torch.zeros(3, 16, 2, 64).to(E4M3),
            "value_cache": torch.zeros(3, 16, 2, 64).to(E4M3), "block_tables": torch.zeros(2, 2, dtype=torch.int32),
            "seq_lens": torch.ones(2, dtype=torch.int32), "softmax_scale": 0.125}
    return args | change


def test_operators_reject_cpu_tensors():
    with pytest.raises(CapabilityError):
        H.paged_decode_attention(**_decode_args())
    with pytest.raises(ValueError, match="query must be a CUDA tensor"):
        H.paged_decode_attention.kernel(**_decode_args())
    q, starts = torch.zeros(4, 2, 64, dtype=BF16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(CapabilityError):
        H.varlen_attention(q, q, q, starts, starts, 0.125)
    with pytest.raises(ValueError, match="query must be a CUDA tensor"):
        H.varlen_attention.kernel(q, q, q, starts, starts, 0.125)
    x = torch.zeros(4, 256, dtype=BF16)
    with pytest.raises(CapabilityError):
        H.rms_norm_quant_fp8(x, x[0], 1e-6)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        H.add_rms_norm_quant_fp8.kernel(x, x, x[0], 1e-6)
    with pytest.raises(TypeError, match="x must have dtype"):
        H.rms_norm_quant_fp8.kernel(x.to(torch.int32), x[0], 1e-6)


def test_meta_kernels_give_output_shapes():
    ops = torch.ops.ayaka
    meta = {k: v.to("meta") if isinstance(v, torch.Tensor) else v for k, v in _decode_args().items()}
    out = ops.paged_decode_attention(**meta)
    assert out.shape == (2, 4, 64) and out.dtype is BF16
    q, k = torch.empty(9, 4, 64, dtype=BF16, device="meta"), torch.empty(20, 2, 64, dtype=BF16, device="meta")
    starts = torch.empty(3, dtype=torch.int32, device="meta")
    assert ops.varlen_attention(q, k, k, starts, starts, 0.1).shape == (9, 4, 64)
    x, w = torch.empty(2, 3, 256, dtype=BF16, device="meta"), torch.empty(256, device="meta")
    q, s = ops.rms_norm_quant_fp8(x, w, 1e-6)
    assert q.shape == (6, 256) and q.dtype is E4M3 and s.shape == (6,) and s.dtype is torch.float32
    q, s, r = ops.add_rms_norm_quant_fp8(x, x, w, 1e-6, 128)
    assert s.shape == (6, 2) and r.shape == x.shape and r.dtype is BF16
    q, s, r = ops.add_rms_norm_quant_fp8(x, x, w, 1e-6, 32, "e8m0", True)
    assert s.shape == (8, 6) and s.dtype is torch.uint8


def test_outputs_keep_the_strides_that_the_meta_kernels_say():
    q = torch.empty(9, 64, 4, dtype=BF16, device="meta").transpose(1, 2)
    starts = torch.empty(3, dtype=torch.int32, device="meta")
    assert torch.ops.ayaka.varlen_attention(q, q, q, starts, starts, 0.1).is_contiguous()


def _paged(**change):
    a = {"q": 1, "dt": _lib.AYK_BF16, "qr": 256, "qh": 64, "kc": 1, "vc": 1, "ct": _lib.AYK_E4M3, "pages": 3, "page": 16,
         "table": 1, "ts": 2, "tw": 2, "lens": 1, "batch": 2, "heads": 4, "kv": 2, "dim": 64, "scale": 0.1, "ks": 1.0,
         "vs": 1.0, "window": 0, "sinks": 0, "out": 1, "ws": None, "wb": 0, "stream": None}
    return _lib.load_library().ayk_paged_decode_attention(*(a | change).values())


def _varlen(**change):
    a = {"q": 1, "qr": 256, "qh": 64, "k": 1, "kr": 128, "kh": 64, "v": 1, "vr": 128, "vh": 64, "dt": _lib.AYK_BF16, "sq": 1,
         "sk": 1, "batch": 2, "tq": 9, "tk": 9, "heads": 4, "kv": 2, "dim": 64, "scale": 0.1, "causal": 1, "window": 0,
         "sinks": 0, "out": 1, "stream": None}
    return _lib.load_library().ayk_varlen_attention(*(a | change).values())


def _norm(**change):
    a = {"x": 1, "dt": _lib.AYK_BF16, "rows": 4, "k": 256, "ldx": 256, "res": None, "ldr": 0, "w": 1, "wt": _lib.AYK_BF16,
         "eps": 1e-6, "group": 0, "st": _lib.AYK_F32, "q": 1, "scale": 1, "srs": 2, "sgs": 1, "ro": None, "stream": None}
    return _lib.load_library().ayk_rms_norm_quant_fp8(*(a | change).values())


@pytest.mark.parametrize("call,change,fragment", [
    (_paged, {"dt": _lib.AYK_F32}, b"query must be"), (_paged, {"ct": _lib.AYK_F32}, b"the cache must be"),
    (_paged, {"ct": _lib.AYK_F16}, b"query's dtype"), (_paged, {"heads": 3}, b"bad shape"), (_paged, {"dim": 257}, b"bad shape"),
    (_paged, {"dim": 0}, b"bad shape"), (_paged, {"kv": 0}, b"bad shape"), (_paged, {"batch": -1}, b"bad shape"),
    (_paged, {"page": 0}, b"bad strides"), (_paged, {"pages": -1}, b"bad strides"), (_paged, {"tw": -1}, b"bad strides"),
    (_paged, {"window": -1}, b"window and sinks"), (_paged, {"sinks": -1}, b"window and sinks"),
    (_paged, {"scale": float("nan")}, b"scales must be finite"), (_paged, {"ks": 0.0}, b"scales must be finite"),
    (_paged, {"vs": float("inf")}, b"scales must be finite"), (_paged, {"heads": 65536, "kv": 1}, b"exceed the grid"),
    (_paged, {"batch": 2**31}, b"exceed the grid"), (_paged, {"q": None}, b"missing operand"), (_paged, {"table": None}, b"missing"),
    (_paged, {"lens": None}, b"missing operand"), (_paged, {"kc": None}, b"missing operand"),
    (_varlen, {"dt": _lib.AYK_E4M3}, b"operands must be"), (_varlen, {"heads": 5}, b"bad shape"), (_varlen, {"dim": 300}, b"bad shape"),
    (_varlen, {"tk": -1}, b"bad shape"), (_varlen, {"kr": -1}, b"strides"), (_varlen, {"window": 4, "causal": 0}, b"needs causal"),
    (_varlen, {"window": -4}, b"window and sinks"), (_varlen, {"scale": float("inf")}, b"scale must be finite"),
    (_varlen, {"tq": 2**31}, b"exceed the grid"), (_varlen, {"batch": 0}, b"without a sequence"), (_varlen, {"k": None}, b"missing"),
    (_norm, {"dt": _lib.AYK_E4M3}, b"x dtype"), (_norm, {"wt": _lib.AYK_U8}, b"weight dtype"), (_norm, {"st": _lib.AYK_BF16}, b"UE8M0 bytes"),
    (_norm, {"k": 0}, b"bad shape"), (_norm, {"ldx": 255}, b"bad shape"), (_norm, {"group": 100}, b"bad shape"),
    (_norm, {"group": -1}, b"bad shape"), (_norm, {"st": _lib.AYK_U8}, b"need a group"), (_norm, {"eps": -1.0}, b"eps must be"),
    (_norm, {"eps": float("nan")}, b"eps must be"), (_norm, {"res": 1, "ldr": 256}, b"come together"), (_norm, {"ro": 1}, b"come together"),
    (_norm, {"group": 128, "srs": 1, "sgs": 1}, b"scale strides"), (_norm, {"rows": 2**31, "group": 0}, b"exceeds the grid"),
    (_norm, {"w": None}, b"missing operand"), (_norm, {"q": None}, b"missing operand"),
])
def test_c_entries_refuse(call, change, fragment):
    assert call(**change) == _lib.AYK_EINVAL
    assert fragment in _lib.load_library().ayk_last_error()


def test_c_entries_with_nothing_to_do():
    assert _paged(batch=0) == _lib.AYK_OK
    assert _varlen(tq=0) == _lib.AYK_OK
    assert _norm(rows=0) == _lib.AYK_OK


def test_definitions_against_torch():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(20, h, 32, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    starts = torch.tensor([0, 20])
    for causal in (True, False):
        got, _ = ora.varlen_attention(q, k, v, starts, starts, 0.3, causal)
        want = torch.nn.functional.scaled_dot_product_attention(
            q.transpose(0, 1), k.repeat_interleave(2, 1).transpose(0, 1), v.repeat_interleave(2, 1).transpose(0, 1),
            is_causal=causal, scale=0.3).transpose(0, 1)
        assert (got - want).abs().max() < 1e-12
    # the last query of a prompt is the decode of its cache
    for window, sinks in ((0, 0), (6, 2)):
        full, _ = ora.varlen_attention(q, k, v, starts, starts, 0.3, True, window, sinks)
        cache = torch.zeros(6, 4, 2, 32, dtype=torch.float64), torch.zeros(6, 4, 2, 32, dtype=torch.float64)
        table = torch.tensor([[4, 1, 0, 5, 2]], dtype=torch.int32)
        for j in range(20):
            cache[0][table[0, j // 4], j % 4], cache[1][table[0, j // 4], j % 4] = k[j], v[j]
        got, _ = ora.paged_decode_attention(q[-1:], *cache, table, torch.tensor([20]), 0.3, window=window, sinks=sinks)
        assert (got - full[-1:]).abs().max() < 1e-12
    x, w = torch.randn(3, 64, generator=g), torch.randn(64, generator=g)
    _, y = ora.rms_norm(x, None, w, 1e-5)
    assert (y - torch.nn.functional.rms_norm(x.double(), (64,), w.double(), 1e-5)).abs().max() < 1e-12
