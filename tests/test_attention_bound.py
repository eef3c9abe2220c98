"""The bound that attention is held to (tests/attention_bound.py), on the CPU: weights rounded as the kernel rounds them are within it, weights of fewer bits
or in the wrong unit are not."""
import pytest

torch = pytest.importorskip("torch")
from tests import attention_bound, attention_cases as cases

F16, BF16 = torch.float16, torch.bfloat16


def _worst(call, **how):
    want, slack = attention_bound.bound(*call)
    return float(((attention_bound.emulate(*call, **how) - want).abs() / slack).max())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_as_the_kernel_rounds(dtype):
    calls = [cases.two_halves(2, 64, 64, 16, dtype), cases.mixed(1, 4, 64, 16, [200, 77], [60, 1], 12, dtype)]
    calls += [cases.unseen(1, 4, 64, 16, 100, 40, 2.0 ** 20, dtype), cases.weightless(1, 4, 64, 16, [150], [30], 2.0 ** 20, dtype, (3, 50))]
    for call in calls:
        assert _worst(call) <= 1


def test_weights_of_fewer_bits():
    assert _worst(cases.two_halves(2, 64, 64, 16, F16), parts=1) > 1
    assert _worst(cases.two_halves(2, 64, 64, 16, BF16), round_to=BF16) > 1


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_weights_in_units_of_the_largest_scale(dtype):
    """whatever weight its token has, and whether or not a row sees it"""
    assert _worst(cases.unseen(1, 4, 64, 16, 100, 40, 2.0 ** 20, dtype), by_scale=True) > 1
    assert _worst(cases.weightless(1, 4, 64, 16, [150], [30], 2.0 ** 20, dtype, (3, 50)), by_scale=True) > 1
