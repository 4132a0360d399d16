"""What the block operators keep of the bits that their inputs and sums have, on the GPU against 64-bit plain forms.

Tolerances, from the arithmetic:
  means       2^-24 of the mean for its rounding, 7 * 2^-24 of the mean magnitude for the seven fp32 additions of a run of
              eight rows, 2^-149 where the mean is below fp32's normal numbers
  attention   CUDA cores: 2^-8 of the result for its one bf16 rounding; 2^-12 of sum p |v| for fp32 scores (a 128-long dot
              product times scale, |s| < 16: 2^-13), exponentials (2^-21) and sums. No term for the probabilities.
"""
import pytest
import torch

import block_ops_ref as ref
from test_gpu_block_ops import AUTO, D, GENERIC, done, lib, ptr, random_lists, randn, run_attention    # noqa: F401

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


def block_means(lib, x, heads, block, mask=None):
    seq, hd = x.shape[0], x.shape[1] // heads
    n = -(-seq // block)
    out, counts, dx = torch.empty(n, heads, hd).cuda(), torch.empty(n, dtype=torch.int32).cuda(), x.cuda()
    dm = None if mask is None else mask.cuda()
    assert lib.iris_b200_block_means(ptr(out), ptr(counts), ptr(dx), heads * hd, seq, heads, hd, block, ptr(dm)) == 0
    done(lib)
    want, wc, mag = ref.means(x, heads, hd, block, mask)
    assert torch.equal(counts.cpu(), wc)
    return out.cpu().double(), want, mag


@pytest.mark.parametrize("hd", [128, 7])
@pytest.mark.parametrize("seq,block", [(1, 64), (64, 64), (333, 128), (1000, 1000), (97, 10)])
@pytest.mark.parametrize("exponent", [0, 127, 124, -126, -133])
def test_block_means_over_the_range_of_bf16(lib, seq, block, hd, exponent):
    """Rows at either end of bf16's range: a sum of eight of the largest has no fp32 value, their mean has."""
    gen = torch.Generator().manual_seed(seq + hd)
    x = torch.randint(-255, 256, (seq, 2 * hd), generator=gen).double() / 128.0            # eight bits, at most 255 / 128
    if exponent > 0:
        x[:, ::2] = x[:, ::2].abs().clamp(min=1.0)          # sums that grow
    x = (x * 2.0 ** exponent).to(torch.bfloat16)
    assert x.isfinite().all() and x.abs().max() > 0
    mask = None if seq < 90 else (torch.arange(seq) % 5 != 0).int()
    got, want, mag = block_means(lib, x, 2, block, mask)
    assert got.isfinite().all()
    assert ((got - want).abs() <= 2.0 ** -24 * want.abs() + 7 * 2.0 ** -24 * mag + 2.0 ** -149).all()


@pytest.mark.parametrize("seq,block", [(4097, 512), (16384, 16384), (3000, 128)])
def test_block_means_of_long_blocks(lib, seq, block):
    """Long sums stay within the error of runs of eight rows."""
    x = (randn(seq, seq, 3 * D) + 40.0).bfloat16()
    got, want, mag = block_means(lib, x, 3, block)
    assert ((got - want).abs() <= 2.0 ** -24 * want.abs() + 7 * 2.0 ** -24 * mag).all()
