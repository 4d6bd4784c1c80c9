"""The numerical tests of test_moe.py under a comparison that NaN cannot pass.  Its own asks whether |got - want| is above the bound, which no NaN is; this one
asks whether it is within.  Same inputs, same bounds; test_expert_gemm_after_a_call_full_of_nan and the NaN weights of test_combine only bite here."""
import math

import pytest

torch = pytest.importorskip("torch")

import test_moe  # noqa: E402
from test_moe import (test_combine, test_expert_gemm_after_a_call_full_of_nan, test_expert_gemm_formats, test_expert_gemm_of_many_experts,  # noqa: E402, F401
                      test_expert_gemm_pitch_of_weights_and_odd_gates, test_expert_gemm_ragged, test_expert_gemm_ranges, test_expert_gemm_sizes_on_gpu,
                      test_expert_gemm_strides_and_values, test_expert_gemm_takes_bad_plans, test_layer)


def check(got, want, off):
    rounded = want.to(got.dtype)
    assert not want.isnan().any() and not off.isnan().any(), "the plain form has no value to compare with"
    over = rounded.isinf()   # above the largest bf16: infinity is the result
    bad = ~torch.where(over, got == rounded, (got.double() - want).abs() <= off)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} too far off, first at {bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]} +- {off[bad][0]}"


@pytest.fixture(autouse=True)
def _strict(monkeypatch):
    monkeypatch.setattr(test_moe, "check", check)


def test_check_wants_numbers():
    want, off = torch.tensor([1.0, -2.0, 0.0, 1e39], dtype=torch.float64), torch.full((4,), 2.0 ** -8, dtype=torch.float64)
    good = torch.tensor([1.0, -2.0, 0.0, math.inf]).bfloat16()
    check(good, want, off)
    for place, value in ((0, math.nan), (1, math.inf), (2, -math.inf), (2, 0.01), (3, math.nan), (3, -math.inf), (3, 1.0)):
        bad = good.clone()
        bad[place] = value
        with pytest.raises(AssertionError):
            check(bad, want, off)
    with pytest.raises(AssertionError):
        check(good, want * math.nan, off)
