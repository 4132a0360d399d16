"""What the block operators keep of the bits that their inputs and sums have, on the GPU against 64-bit plain forms.

Tolerances, from the arithmetic:
  attention   CUDA cores: 2^-8 of the result for its one bf16 rounding; 2^-12 of sum p |v| for fp32 scores (a 128-long dot
              product times scale, |s| < 16: 2^-13), exponentials (2^-21) and sums. No term for the probabilities.
"""
import pytest
import torch

import block_ops_ref as ref
from test_gpu_block_ops import AUTO, GENERIC, lib, random_lists, randn, run_attention    # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel,q_block,k_block", [(GENERIC, 100, 3), (GENERIC, 1, 3), (AUTO, 100, 3), (AUTO, 1, 3)])
@pytest.mark.parametrize("hd", [64, 128])
def test_probabilities_keep_fp32_on_the_cuda_cores(lib, kernel, q_block, k_block, hd):
    """Few keys a row, so that the rounding of a probability to bf16 would be of the size of the results."""
    sq, sk, heads = 200, 60, 2
    q, k, v = (randn(i, r, c).bfloat16() for i, (r, c) in enumerate([(sq, heads * hd), (sk, hd), (sk, hd)]))
    lists = random_lists(5, heads, -(-sq // q_block), sk // k_block, 2)
    got = run_attention(lib, q, k, v, heads, 1, hd, None, lists, q_block, k_block, kernel)
    want, mag = ref.attention(q, k, v, heads, 1, hd, hd ** -0.5, None, lists, q_block, k_block)
    assert ((got - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -12 * mag)).max().item() <= 0.0
