"""CPU tests of the context attention ops' arguments at the ends of their range."""
import pytest
import torch

from semicat_amd import RelativeBias, context_backward, context_forward, relative_bucket_starts
from tests.test_context import _t


def test_the_statistics_of_a_row_are_two_numbers():
    q = _t(1, 2, 3, 32)
    for shape in ((1, 2, 3), (1, 2, 3, 1), (2, 1, 2, 3)):
        with pytest.raises(AssertionError):
            context_backward(q, q, q, q, _t(*shape, dtype=torch.float32), q)


@pytest.mark.parametrize("start", [1.5, 2.0, "1", None])
def test_query_start_is_a_whole_number(start):
    with pytest.raises(TypeError):
        context_forward(*[_t(1, 2, 3, 32)] * 3, query_start=start)


@pytest.mark.parametrize("call", [lambda: relative_bucket_starts(16, 100.5), lambda: relative_bucket_starts(16.0, 128),
                                  lambda: relative_bucket_starts(16, 128.0), lambda: RelativeBias(_t(32, 2), 128.0)])
def test_buckets_and_distances_are_whole_numbers(call):
    """Also where a whole number of the same value was asked for before."""
    relative_bucket_starts(16, 128)
    with pytest.raises(TypeError):
        call()
