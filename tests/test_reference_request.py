"""CPU: the request for reference operators is read from the environment as it stands."""

import os

import pytest
import torch

import ayaka.kernel.hip as H
from ayaka.utils.import_utils import CapabilityError


def _refused():
    with pytest.raises(CapabilityError) as info:
        H.per_token_quant_fp8(torch.zeros(2, 64))
    return "no plain-torch reference mode" in str(info.value)


def test_a_replaced_environment_counts(monkeypatch):
    assert not _refused()  # a CPU tensor is refused for being one
    monkeypatch.setattr(os, "environ", {**os.environ, "AYAKA_FORCE_REFERENCE_OPS": "1"})
    assert _refused()


@pytest.mark.parametrize("value,asked", [("1", True), ("TRUE", True), ("yes", True), ("0", False), ("", False)])
def test_a_set_variable_counts(monkeypatch, value, asked):
    monkeypatch.setenv("AYAKA_FORCE_REFERENCE_OPS", value)
    assert _refused() is asked
