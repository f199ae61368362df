"""Calls whose rows have as many parts as there can be for so many keys: all of them are made.  Tolerances: test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,q,k,n", [(torch.float32, 16, 513, 5), (torch.float32, 16, 1025, 3), (torch.float32, 1, 513, 40),
                                         (torch.float32, 3, 2049, 2), (torch.bfloat16, 7, 513, 6), (torch.bfloat16, 7, 1025, 4),
                                         (torch.bfloat16, 16, 4097, 2), (torch.float16, 8, 4097, 2), (torch.bfloat16, 1, 1025, 9)])
@pytest.mark.parametrize("causal", [False, True])
def test_as_many_parts_as_there_can_be(ops, dtype, q, k, n, causal):
    check(ops, *make([q] * n, [k] * n, 2, 1, 32, dtype), [q] * n, [k] * n, causal)


def test_different_ones_together(ops):
    q_lens, k_lens = [16, 7, 1, 16, 7, 3], [4097, 513, 1025, 5121, 4096, 513]
    check(ops, *make(q_lens, k_lens, 4, 2, 64, torch.bfloat16), q_lens, k_lens, False)
    check(ops, *make(q_lens, k_lens, 4, 2, 64, torch.float32), q_lens, k_lens, True)
