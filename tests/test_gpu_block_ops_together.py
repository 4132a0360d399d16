"""The block operators side by side and over and over: every call of every round into buffers of its own, that hold nothing
right beforehand, against what the same call gives alone; and single rows of a cache whose offsets pass 32 bits."""
import pytest
import torch

import block_ops_ref as ref
from test_gpu_block_ops import AUTO, D, TCGEN05, done, lib, ptr, randn      # noqa: F401 (lib is a fixture)

pytestmark = pytest.mark.gpu

HEADS, SEQ, QB, KB, N = 16, 4000, 128, 64, 9
NQ, NK, W = -(-SEQ // QB), -(-SEQ // KB), HEADS * D


class Inputs:
    def __init__(self, seed):
        self.q, self.k, self.v = (randn(seed + i, SEQ, W).bfloat16().cuda() for i in range(3))
        gen = torch.Generator().manual_seed(seed)
        # the last query tiles of the CTAs have no keys; the others one block
        self.sparse = torch.full((HEADS, NQ, N), -1, dtype=torch.int32)
        some = torch.rand(HEADS, NQ, generator=gen) < 0.4
        some.view(-1)[-300:] = False
        self.sparse[..., 2][some] = torch.randint(0, NK, (int(some.sum()),), generator=gen, dtype=torch.int32)
        self.sparse = self.sparse.cuda()


class Buffers:
    def __init__(self):
        self.qm, self.km = (torch.full((n, HEADS, D), float("nan"), device="cuda") for n in (NQ, NK))
        self.lists = torch.full((HEADS, NQ, N), -1, dtype=torch.int32, device="cuda")
        self.out = torch.full((SEQ, W), float("nan"), dtype=torch.bfloat16, device="cuda")

    def same(self, other):
        return all(torch.equal(a.nan_to_num(7.25), b.nan_to_num(7.25)) for a, b in
                   ((self.qm, other.qm), (self.km, other.km), (self.lists, other.lists), (self.out, other.out)))


def attend(lib, x, b, lists, rows, q_block, kernel):
    return lib.iris_b200_attention_blocks(ptr(b.out), W, ptr(x.q), W, ptr(x.k), W, ptr(x.v), W, rows, SEQ, HEADS, HEADS, D, D ** -0.5,
                                          None, ptr(lists), N, q_block, KB, kernel)


def chain(lib, x, b):
    rc = lib.iris_b200_block_means(ptr(b.qm), None, ptr(x.q), W, SEQ, HEADS, D, QB, None)
    rc |= lib.iris_b200_block_means(ptr(b.km), None, ptr(x.k), W, SEQ, HEADS, D, KB, None)
    rc |= lib.iris_b200_block_select(ptr(b.lists), ptr(b.qm), ptr(b.km), None, NQ, NK, HEADS, HEADS, D, N, 1, 0)
    return rc | attend(lib, x, b, b.lists, SEQ, QB, TCGEN05)


def rows(lib, x, b):
    rc = lib.iris_b200_block_means(ptr(b.qm), None, ptr(x.q), W, 1, HEADS, D, 1, None)
    rc |= lib.iris_b200_block_means(ptr(b.km), None, ptr(x.k), W, SEQ, HEADS, D, KB, None)
    rc |= lib.iris_b200_block_select(ptr(b.lists), ptr(b.qm), ptr(b.km), None, 1, NK, HEADS, HEADS, D, N, 0, 0)
    return rc | attend(lib, x, b, b.lists, 1, 1, AUTO)


def sparse(lib, x, b):
    return attend(lib, x, b, x.sparse, SEQ, QB, TCGEN05)


def dense(lib, x, b):
    return lib.iris_b200_attention_ex(ptr(b.out), W, ptr(x.q), ptr(x.k), ptr(x.v), W, SEQ, SEQ, HEADS, HEADS, D, D ** -0.5, 0, None, 0)


@pytest.mark.parametrize("what", [(chain, chain, rows, dense), (sparse, sparse, chain, rows), (sparse, chain, sparse, dense)])
def test_every_round_of_calls_on_several_streams(lib, what):
    home, side = torch.cuda.current_stream(), [torch.cuda.Stream() for _ in what]
    inputs = [Inputs(10 * i) for i in range(len(what))]
    alone = [Buffers() for _ in what]
    for fn, x, b in zip(what, inputs, alone):
        assert fn(lib, x, b) == 0
        done(lib)
    rounds = [[Buffers() for _ in what] for _ in range(10)]
    torch.cuda.synchronize()
    try:
        for r in rounds:
            for fn, x, b, s in zip(what, inputs, r, side):
                assert lib.iris_b200_use_stream(s.cuda_stream) == 0
                assert fn(lib, x, b) == 0
        torch.cuda.synchronize()
    finally:
        lib.iris_b200_use_stream(home.cuda_stream)
    done(lib)
    for n, r in enumerate(rounds):
        for i, (b, a) in enumerate(zip(r, alone)):
            assert b.same(a), (n, i)
    for i, fn in enumerate(what):            # what they are compared with is not what they began with
        first = SEQ if fn is not rows else 1
        assert alone[i].out[:first].isfinite().all() and alone[i].out[first:].isnan().all()


def test_a_call_repeats_itself_to_the_bit(lib):
    """Full lists, lists of different lengths with a mask, a list cut over a cluster, single rows; other calls in between."""
    x = Inputs(77)
    mask = (torch.rand(SEQ, generator=torch.Generator().manual_seed(1)) < 0.9).int().cuda()
    full = torch.rand(HEADS, NQ, NK, device="cuda").argsort(2)[:, :, :N].sort(2)[0].int().contiguous()
    short = full.clone()
    short[torch.rand(HEADS, NQ, N, device="cuda") < 0.3] = -1
    cases = [(full, None, SEQ, QB, TCGEN05), (short, mask, SEQ, QB, TCGEN05), (full, mask, 100, QB, TCGEN05), (short, mask, 1, 1, AUTO)]

    def run(lists, m, n, qb, kernel):
        out = torch.full((SEQ, W), 7.0, dtype=torch.bfloat16, device="cuda")
        lists = lists[:, :-(-n // qb)].contiguous()
        assert lib.iris_b200_attention_blocks(ptr(out), W, ptr(x.q), W, ptr(x.k), W, ptr(x.v), W, n, SEQ, HEADS, HEADS, D, D ** -0.5,
                                              ptr(m), ptr(lists), N, qb, KB, kernel) == 0
        return out

    first = [run(*c) for c in cases]
    for _ in range(20):
        again = [run(*c) for c in cases]
        done(lib)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_single_rows_of_a_cache_whose_offsets_pass_32_bits(lib, hd):
    """K and V in one tensor, V behind K in a row; the first and the last block, and one on either side of 2^31 elements."""
    seq, ld, kb = 262400, 8320, 64
    x = torch.empty(seq, ld, dtype=torch.bfloat16, device="cuda")
    x[:, :2 * hd] = randn(1, seq, 2 * hd).bfloat16().cuda()
    middle = 2 ** 31 // ld // kb
    assert seq * ld > 2 ** 31 + 2 ** 25 and (middle + 1) * kb * ld > 2 ** 31 > middle * kb * ld
    blocks = [0, middle - 1, middle, middle + 1, seq // kb - 1]
    lists = torch.tensor([[blocks, blocks[::-1]]], dtype=torch.int32)          # two rows
    keys = torch.cat([torch.arange(b * kb, b * kb + kb) for b in blocks]).cuda()
    k, v = x[keys, :hd].cpu(), x[keys, hd:2 * hd].cpu()
    q = randn(2, 2, hd).bfloat16()
    want, mag = ref.attention(q, k, v, 1, 1, hd, hd ** -0.5, None, torch.arange(5).expand(1, 2, 5), 1, kb)
    dq, dl = q.cuda(), lists.cuda()
    for n in (2, 1):
        out = torch.full((3, hd), 7.0, dtype=torch.bfloat16, device="cuda")
        dn = dl[:, :n].contiguous()
        assert lib.iris_b200_attention_blocks(ptr(out), hd, ptr(dq), hd, ptr(x), ld, ptr(x, hd), ld, n, seq, 1, 1, hd, hd ** -0.5, None,
                                              ptr(dn), 5, 1, kb, AUTO) == 0
        done(lib)
        got = out[:n].cpu().double()
        # fp32 scores of up to 256 dimensions: 2^-12; the result is rounded once
        assert ((got - want[:n]).abs() <= 2.0 ** -8 * want[:n].abs() + 2.0 ** -12 * mag[:n]).all()
        assert (out[n:] == 7).all()
