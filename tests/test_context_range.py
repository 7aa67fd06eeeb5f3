"""CPU tests of the context attention ops' arguments at the ends of their range."""
import pytest
import torch

from semicat_amd import context_backward
from tests.test_context import _t


def test_the_statistics_of_a_row_are_two_numbers():
    q = _t(1, 2, 3, 32)
    for shape in ((1, 2, 3), (1, 2, 3, 1), (2, 1, 2, 3)):
        with pytest.raises(AssertionError):
            context_backward(q, q, q, q, _t(*shape, dtype=torch.float32), q)
