"""Without a GPU: refusals, meta kernels and C argument checks of the rotation, the 4-bit cache, its
attention and the MoE layer for few tokens."""

import pytest
import torch

import ayaka.kernel.hip as H
from ayaka.kernel.hip import _lib
from ayaka.utils.import_utils import CapabilityError
from tests._decode_step import decode_case, moe_case, mx_planes, table

BF16 = torch.bfloat16
PLANES = ("key_codes", "key_scales", "value_codes", "value_scales")


def _rope_args():
    q, k = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(3, 2, 64, dtype=BF16)
    return {"query": q, "key": k, "value": k, "positions": torch.zeros(3, dtype=torch.int64), "cos_sin": table(8, 64),
            "slots": torch.zeros(3, dtype=torch.int64), "query_out": torch.zeros_like(q)}


def _calls():
    planes = dict(zip(PLANES, (*mx_planes(2, 2, 16, 64, 0), *mx_planes(2, 2, 16, 64, 1))))
    cache = torch.zeros(2, 16, 2, 64, dtype=BF16)
    rope = _rope_args()
    c = decode_case([3, 9], 4, 2, 64, 16)
    return {
        H.rope_write_kv: rope | {"key_cache": cache, "value_cache": cache, "k_inverse": 1.0, "v_inverse": 1.0},
        H.rope_write_kv_mxfp4: rope | planes,
        H.write_kv_mxfp4: {n: rope[n] for n in ("key", "value", "slots")} | planes,
        H.gather_cache_mxfp4: {"codes": planes["key_codes"], "scales": planes["key_scales"], "slots": rope["slots"],
                               "destination": torch.zeros(3, 2, 64)},
        H.paged_decode_attention_mxfp4: {n: c[n] for n in ("query", *PLANES, "block_tables", "seq_lens")} | {"softmax_scale": 0.1},
        H.fp8_block_moe_small: moe_case(3, 4, 2, 256, 128),
    }


def test_operators_reject_cpu_tensors():
    for op, args in _calls().items():
        with pytest.raises(CapabilityError):
            op(**args)
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            op.kernel(**args)


def test_meta_kernels_give_output_shapes():
    for op, args in _calls().items():
        meta = {k: v.to("meta") if isinstance(v, torch.Tensor) else v for k, v in args.items()}
        out = getattr(torch.ops.ayaka, op.name)(**meta)
        if op in (H.paged_decode_attention_mxfp4, H.fp8_block_moe_small):
            like = meta["query"] if "query" in meta else meta["x"]
            assert out.shape == like.shape and out.dtype is like.dtype and out.is_contiguous()
        else:
            assert out is None


def _rope(**change):
    a = {"q": 1, "qr": 256, "qh": 64, "k": 1, "kr": 128, "kh": 64, "v": 1, "vr": 128, "vh": 64, "dt": _lib.AYK_BF16, "tokens": 3,
         "heads": 4, "kv": 2, "dim": 64, "pos": 1, "table": 1, "tr": 8, "rotary": 64, "side": 0, "qo": 1, "qor": 256, "qoh": 64,
         "ko": None, "kor": 0, "koh": 0, "kc": 1, "vc": 1, "ct": _lib.AYK_E4M3, "n": 32, "slots": 1, "ki": 1.0, "vi": 1.0, "st": None}
    return _lib.load_library().ayk_rope_kv_write(*(a | change).values())


def _rope4(**change):
    a = {"q": 1, "qr": 256, "qh": 64, "k": 1, "kr": 128, "kh": 64, "v": 1, "vr": 128, "vh": 64, "dt": _lib.AYK_BF16, "tokens": 3,
         "heads": 4, "kv": 2, "dim": 64, "pos": 1, "table": 1, "tr": 8, "rotary": 64, "side": 0, "qo": 1, "qor": 256, "qoh": 64,
         "ko": None, "kor": 0, "koh": 0, "kc": 1, "ks": 1, "vc": 1, "vs": 1, "pages": 2, "page": 16, "slots": 1, "st": None}
    return _lib.load_library().ayk_rope_kv_write_mxfp4(*(a | change).values())


def _gather4(**change):
    a = {"c": 4, "s": 4, "pages": 2, "page": 16, "kv": 2, "dim": 64, "slots": 1, "n": 3, "dest": 16, "dt": _lib.AYK_BF16, "st": None}
    return _lib.load_library().ayk_kv_gather_mxfp4(*(a | change).values())


def _decode4(**change):
    a = {"q": 16, "dt": _lib.AYK_BF16, "qr": 256, "qh": 64, "kc": 16, "ks": 16, "vc": 16, "vs": 16, "pages": 3, "page": 16, "table": 4,
         "ts": 2, "tw": 2, "lens": 4, "batch": 2, "heads": 4, "kv": 2, "dim": 64, "scale": 0.1, "window": 0, "sinks": 0, "out": 16,
         "ws": None, "wb": 0, "st": None}
    return _lib.load_library().ayk_paged_decode_attention_mxfp4(*(a | change).values())


def _moe(**change):
    a = {"x": 16, "dt": _lib.AYK_BF16, "ldx": 256, "tokens": 3, "gu": 16, "gs": 4, "dn": 16, "ds": 4, "experts": 4, "hidden": 256,
         "inner": 128, "w": 4, "ids": 4, "topk": 2, "out": 2, "ldo": 256, "ws": 16, "wb": 1 << 20, "st": None}
    return _lib.load_library().ayk_fp8_block_moe_small(*(a | change).values())


@pytest.mark.parametrize("call,change,fragment", [
    *[(call, change, fragment) for call in (_rope, _rope4) for change, fragment in (
        ({"dt": _lib.AYK_F32}, b"must be float16"), ({"tokens": -1}, b"bad shape"), ({"heads": -1}, b"bad shape"),
        ({"kv": 0}, b"bad shape"), ({"dim": 257}, b"bad shape"), ({"dim": 0}, b"bad shape"), ({"rotary": 63}, b"rotated dims"),
        ({"rotary": 66}, b"rotated dims"), ({"rotary": -2}, b"rotated dims"), ({"tr": 0}, b"is empty"), ({"kr": -1}, b"strides"),
        ({"qoh": -1}, b"strides"), ({"tokens": 2**24}, b"too many tokens"), ({"q": None}, b"missing operand"),
        ({"qo": None}, b"missing operand"), ({"v": None}, b"missing operand"), ({"slots": None}, b"missing operand"),
        ({"pos": None}, b"missing operand"), ({"table": None}, b"missing operand"), ({"kc": None}, b"missing operand"))],
    (_rope, {"ct": _lib.AYK_F16}, b"the cache must be"), (_rope, {"ct": _lib.AYK_U8}, b"the cache must be"),
    (_rope, {"n": -1}, b"bad cache"), (_rope, {"ki": 0.0}, b"inverse scales"), (_rope, {"vi": float("inf")}, b"inverse scales"),
    (_rope, {"ki": float("nan")}, b"inverse scales"),
    (_rope4, {"dim": 48, "rotary": 48}, b"multiple of 32"), (_rope4, {"pages": -1}, b"bad cache"), (_rope4, {"page": 0}, b"bad cache"),
    (_rope4, {"vs": None}, b"missing operand"),
    (_gather4, {"n": -1}, b"bad shape"), (_gather4, {"dim": 40}, b"bad shape"), (_gather4, {"dim": 288}, b"bad shape"),
    (_gather4, {"kv": 0}, b"bad shape"), (_gather4, {"page": 0}, b"bad shape"), (_gather4, {"dt": _lib.AYK_E4M3}, b"destination"),
    (_gather4, {"slots": None}, b"missing"), (_gather4, {"c": None}, b"missing"), (_gather4, {"c": 2}, b"aligned"),
    (_gather4, {"n": 2**31}, b"too many rows"),
    (_decode4, {"dt": _lib.AYK_F32}, b"query must be"), (_decode4, {"heads": 3}, b"bad shape"), (_decode4, {"dim": 72}, b"bad shape"),
    (_decode4, {"dim": 288}, b"bad shape"), (_decode4, {"batch": -1}, b"bad shape"), (_decode4, {"page": 12}, b"bad strides"),
    (_decode4, {"page": 0}, b"bad strides"), (_decode4, {"pages": -1}, b"bad strides"), (_decode4, {"tw": -1}, b"bad strides"),
    (_decode4, {"qr": -1}, b"bad strides"), (_decode4, {"window": -1}, b"window and sinks"), (_decode4, {"sinks": -1}, b"window and sinks"),
    (_decode4, {"scale": float("nan")}, b"must be finite"), (_decode4, {"tw": 2**27}, b"positions"), (_decode4, {"pages": 2**27}, b"rows of a head"),
    (_decode4, {"heads": 65536}, b"exceed the grid"), (_decode4, {"batch": 2**24}, b"exceed the grid"),
    (_decode4, {"q": None}, b"missing operand"), (_decode4, {"table": None}, b"missing operand"), (_decode4, {"vs": None}, b"missing operand"),
    (_decode4, {"vc": 8}, b"aligned"), (_decode4, {"out": 2}, b"aligned"),
    (_moe, {"dt": _lib.AYK_F32}, b"x must be"), (_moe, {"tokens": 65}, b"at most 64 tokens"), (_moe, {"tokens": -1}, b"at most 64"),
    (_moe, {"experts": 0}, b"1 to 1024 experts"), (_moe, {"experts": 1025}, b"1 to 1024 experts"), (_moe, {"hidden": 192}, b"multiples of 128"),
    (_moe, {"inner": 64}, b"multiples of 128"), (_moe, {"inner": 0}, b"multiples of 128"), (_moe, {"topk": 0}, b"bad topk"),
    (_moe, {"ldx": 128}, b"row strides"), (_moe, {"ldo": 255}, b"row strides"), (_moe, {"x": None}, b"missing operand"),
    (_moe, {"ids": None}, b"missing operand"), (_moe, {"ldx": 260}, b"aligned"), (_moe, {"dn": 8}, b"aligned"),
])
def test_c_entries_refuse(call, change, fragment):
    assert call(**change) == _lib.AYK_EINVAL
    assert fragment in _lib.load_library().ayk_last_error()


def test_c_entries_with_nothing_to_do():
    assert _rope(tokens=0) == _lib.AYK_OK
    assert _rope4(tokens=0) == _lib.AYK_OK
    assert _gather4(n=0) == _lib.AYK_OK
    assert _decode4(batch=0) == _lib.AYK_OK
    assert _moe(tokens=0) == _lib.AYK_OK


def test_workspaces():
    for change in ({"ws": None}, {"ws": 8}, {"wb": 1}):
        assert _moe(**change) == _lib.AYK_EWORKSPACE
    moe = lambda *a: _lib.query("ayk_fp8_block_moe_small_scratch_bytes", *a)  # noqa: E731
    # what lies between the projections, four partial results of 56 channel blocks, a counter of each
    assert moe(64, 8, 256, 7168, 2048) == 64 * 8 * 2048 * 4 + 4 * 64 * 7168 * 4 + 56 * 4
    # a row for every expert that a token can name
    assert moe(64, 100, 8, 7168, 2048) - moe(64, 8, 8, 7168, 2048) == 0
    assert moe(1, 1, 1, 128, 128) == 128 * 4 + 128 * 4 + 4
    for bad in ((65, 8, 256, 7168, 2048), (0, 8, 256, 7168, 2048), (64, 0, 256, 7168, 2048), (64, 8, 1025, 7168, 2048),
                (64, 8, 256, 7168, 0), (64, 8, 256, 0, 2048), (64, 8, 256, 2**25, 2048), (64, 2**15, 256, 7168, 2048)):
        assert moe(*bad) == 0
    split = lambda *a: _lib.query("ayk_paged_decode_attention_mxfp4_split_bytes", *a)  # noqa: E731
    for dim, width in ((32, 64), (64, 64), (96, 128), (128, 128), (160, 256)):
        assert split(1, 32, 8, dim, 131072, 0, 0) == 2 * 1024 * 16 * (width + 2) * 4
    assert split(1, 32, 8, 128, 1024, 0, 0) == 0
    assert split(1, 32, 8, 128, 131072, 1024, 4) == 0
    assert split(1, 32, 8, 128, 131072, 2**62, 2**62) > 0
    for bad in ((0, 32, 8, 128, 9, 0, 0), (1, 0, 8, 128, 9, 0, 0), (1, 32, 0, 128, 9, 0, 0), (1, 32, 8, 100, 131072, 0, 0),
                (1, 32, 8, 128, -1, 0, 0), (1, 32, 8, 128, 9, -1, 0), (1, 32, 8, 128, 9, 0, -1)):
        assert split(*bad) == 0
