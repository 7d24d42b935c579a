"""CPU: refusals of the split entry of packed attention, and what the workspace queries answer."""

import pytest

from ayaka.kernel.hip import _lib


def _split(**change):
    a = {"q": 1, "qr": 256, "qh": 64, "k": 1, "kr": 128, "kh": 64, "v": 1, "vr": 128, "vh": 64, "dt": _lib.AYK_BF16, "sq": 1,
         "sk": 1, "batch": 2, "tq": 9, "tk": 9, "heads": 4, "kv": 2, "dim": 64, "scale": 0.1, "causal": 1, "window": 0,
         "sinks": 0, "out": 1, "ws": None, "wb": 0, "stream": None}
    return _lib.load_library().ayk_varlen_attention_split(*(a | change).values())


@pytest.mark.parametrize("change,fragment", [
    ({"dt": _lib.AYK_F32}, b"operands must be"), ({"heads": 5}, b"bad shape"), ({"dim": 257}, b"bad shape"),
    ({"kv": 0}, b"bad shape"), ({"tq": -1}, b"bad shape"), ({"vh": -1}, b"strides"), ({"window": 4, "causal": 0}, b"needs causal"),
    ({"sinks": -4}, b"window and sinks"), ({"scale": float("nan")}, b"scale must be finite"), ({"tk": 2**31}, b"exceed the grid"),
    ({"batch": 0}, b"without a sequence"), ({"v": None}, b"missing"), ({"out": None}, b"missing"),
])
def test_split_entry_refuses(change, fragment):
    assert _split(**change) == _lib.AYK_EINVAL
    assert fragment in _lib.load_library().ayk_last_error()


def test_split_entry_with_nothing_to_do():
    assert _split(tq=0) == _lib.AYK_OK


def test_workspaces_hold_what_the_kernels_write():
    split = lambda *a: _lib.query("ayk_varlen_attention_split_workspace_bytes", *a)  # noqa: E731
    # 512 rows of 32 heads are 128 workgroups: four parts of a row of 128 sums, maximum and sum
    assert split(1, 512, 32, 128) == 4 * 512 * 32 * 132 * 4
    assert split(1, 1, 1, 64) == 16 * 68 * 4  # never more than sixteen parts
    assert split(1, 8192, 64, 128) == 0  # the chip is full
    assert split(300, 300, 2, 64) == 0  # a tile a sequence
    paged = lambda *a: _lib.query("ayk_paged_decode_attention_workspace_bytes", *a)  # noqa: E731
    for dim, width in ((128, 128), (80, 96), (200, 256)):
        assert paged(4, 32, 8, dim) == 2 * 1024 * 16 * (width + 2) * 4
    assert paged(4, 32, 8, 100) == 0  # the row kernel takes none
    assert paged(4, 4, 8, 128) == 0
    # sequences that stay whole ask for none
    split_bytes = lambda *a: _lib.query("ayk_paged_decode_attention_split_bytes", *a)  # noqa: E731
    assert split_bytes(1, 32, 8, 128, _lib.AYK_E4M3, 1024, 0, 0) == 0
    assert split_bytes(1, 32, 8, 128, _lib.AYK_E4M3, 100000, 0, 0) == paged(1, 32, 8, 128)
    assert split_bytes(1, 32, 8, 128, _lib.AYK_E4M3, 100000, 1024, 4) == 0
    assert split_bytes(1, 32, 8, 128, _lib.AYK_E4M3, 100000, 2**62, 2**62) == paged(1, 32, 8, 128)
    assert split_bytes(1, 32, 8, 100, _lib.AYK_BF16, 100000, 0, 0) == 0
    for bad in ((0, 32, 8, 128, 3, 9, 0, 0), (1, 0, 8, 128, 3, 9, 0, 0), (1, 32, 0, 128, 3, 9, 0, 0), (1, 32, 8, 128, 0, 9, 0, 0),
                (1, 32, 8, 128, 3, -1, 0, 0), (1, 32, 8, 128, 3, 9, -1, 0)):
        assert split_bytes(*bad) == 0
