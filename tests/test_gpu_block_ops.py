"""The multi-axis rotation, the block means, the block lists and the attention
over them, on the GPU against 64-bit plain forms (block_ops_ref.py).

Tolerances, all derived from the arithmetic:
  tables      2e-7: the phase is cut to 2^-32 turns (1.5e-9 rad), the angle (<= pi / 4) rounded twice (2 * 2^-24 * 0.79),
              the series within 2e-9, their evaluation and result rounded (about 1.5 * 2^-24)
  prologue    one bf16 rounding (2^-8 of the value) plus, of the magnitudes |a| + |b| that a rotation adds, 2e-7 for the
              angle and 2^-20 for the fp32 norm and products
  means       2^-24 of the mean, and of the mean magnitude 15 * 2^-24 (sums of up to 16 rows in fp32)
  attention   one bf16 rounding of every probability (2^-8 of sum p |v|) and of the result (2^-8 of it); 2^-12 of
              sum p |v| covers fp32 scores (a 128-long dot product times scale, |s| < 16: 2^-13) and exponentials (2^-21)
"""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import block_ops_ref as ref

pytestmark = pytest.mark.gpu

GENERIC, TCGEN05, AUTO = 2, 1, 0
D = 128
NAN = float("nan")


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge
    lib = ge.load_package().load()
    lib.init()
    torch.cuda.set_device(0)
    before, mine = torch.cuda.current_stream(), torch.cuda.Stream()
    torch.cuda.set_stream(mine)              # the library's operations in order with torch's
    assert lib.iris_b200_attach_stream(mine.cuda_stream) == 0
    yield lib
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)
    lib.iris_b200_attach_stream(None)
    lib.check()


def gpu(t):
    return None if t is None else t.cuda()


def ptr(t, offset=0):
    return None if t is None else t.data_ptr() + offset * t.element_size()


def done(lib):
    lib.iris_dev_sync()
    torch.cuda.synchronize()
    lib.check()


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# ---------------------------------------------------------------------------
# rotation
# ---------------------------------------------------------------------------

AXES = [((32, 32, 32, 32), None, 2000.0, False), ((32, 48, 48), (2.5, 1.0, 1.0), 256.0, False),
        ((16, 24, 24), (0.625, 1.0, -1.0), 10000.0, True), ((128,), (24.0,), 1e6, False)]


def positions(seed, seq, n, most=70000):
    return torch.randint(-most, most, (seq, n), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


@pytest.mark.parametrize("seq,hd,axes", [(1, 128, 0), (2, 128, 1), (517, 128, 2), (4096, 128, 3), (33, 130, 2), (7, 64, 2),
                                         (65, 512, 0), (9, 6, 4)])
def test_tables(lib, seq, hd, axes):
    dims, scales, theta, one = (AXES + [((2, 2), None, 10.0, False)])[axes]
    if hd == 64:
        dims = (16, 24, 24)
    n = len(dims)
    plan = lib.rope_axes(dims, scales, theta, one, hd)
    pos = positions(seq, seq, n)
    cos, sin = torch.full((seq + 1, hd // 2), NAN).cuda(), torch.full((seq + 1, hd // 2), NAN).cuda()
    dp = pos.cuda()
    assert lib.iris_b200_rope_axes_tables(ptr(cos), ptr(sin), ptr(dp), plan, seq, hd) == 0
    done(lib)
    ang = ref.angles(pos, dims, scales, theta, one, hd)
    # the 64-bit angle itself is off by 2^-52 of its value
    slack = 2e-7 + ang.abs().max().item() * 2.0 ** -51
    assert (cos[:seq].cpu().double() - ang.cos()).abs().max() <= slack
    assert (sin[:seq].cpu().double() - ang.sin()).abs().max() <= slack
    assert cos[seq].isnan().all() and sin[seq].isnan().all()          # the row behind the last one


def test_tables_extreme_positions(lib):
    """The ends of the int32 range, against integer arithmetic on the plan's own fractions."""
    plan = lib.rope_axes((128,), None, 10000.0, False, 128)
    pos = torch.tensor([[2 ** 31 - 1], [-2 ** 31], [0], [1], [-1]], dtype=torch.int32)
    cos, sin = torch.empty(5, 64).cuda(), torch.empty(5, 64).cuda()
    dp = pos.cuda()
    assert lib.iris_b200_rope_axes_tables(ptr(cos), ptr(sin), ptr(dp), plan, 5, 128) == 0
    done(lib)
    turn = np.array([[(int(p) * plan.turn[j]) % (1 << 64) / 2.0 ** 64 for j in range(64)] for p in pos[:, 0]])
    assert np.abs(cos.cpu().numpy() - np.cos(2 * np.pi * turn)).max() <= 2e-7
    assert np.abs(sin.cpu().numpy() - np.sin(2 * np.pi * turn)).max() <= 2e-7


def prologue(lib, seq, heads, kv, hd, dims, split, norm, in_place=False, pad=0, off=0, q_only=False, seed=1, scales=None,
             theta=10000.0, one=False):
    eps = 1e-6
    plan = lib.rope_axes(dims, scales, theta, one, hd)
    pos = positions(seed, seq, len(dims), 3000)
    width = (heads + kv) * hd
    ldi = width + pad
    x = (randn(seed + 1, seq, ldi) * 1.7).bfloat16()
    wq, wk = (1.0 + 0.25 * randn(3, hd), 1.0 + 0.25 * randn(4, hd)) if norm else (None, None)
    flat = torch.cat([torch.zeros(off).bfloat16(), x.reshape(-1)]).cuda()
    dp, dwq, dwk = pos.cuda(), gpu(wq), gpu(wk)
    q, k = ptr(flat, off), ptr(flat, off + heads * hd)
    ldq, ldk = (ldi, ldi) if in_place else (heads * hd + pad, kv * hd + 2 * pad)
    if in_place:
        qo, ko = q, k
    else:
        bq = torch.full((seq + 1, ldq), 7.0).bfloat16().cuda()
        bk = torch.full((seq + 1, max(ldk, 1)), 7.0).bfloat16().cuda()
        qo, ko = ptr(bq), ptr(bk)
    if q_only:
        rc = lib.iris_b200_qk_norm_rope_axes(qo, ldq, None, 0, q, None, ldi, ptr(dwq), None, ptr(dp), plan, seq, heads, 0, hd, eps,
                                             int(split))
    else:
        rc = lib.iris_b200_qk_norm_rope_axes(qo, ldq, ko, ldk, q, k, ldi, ptr(dwq), ptr(dwk), ptr(dp), plan, seq, heads, kv, hd,
                                             eps, int(split))
    assert rc == 0
    done(lib)
    ang = ref.angles(pos, dims, scales, theta, one, hd)
    wq_y, wq_m = ref.norm_rope(x[:, :heads * hd], heads, hd, wq, eps, ang, split)
    wk_y, wk_m = ref.norm_rope(x[:, heads * hd:width], kv, hd, wk, eps, ang, split) if kv else (None, None)

    def close(got, want, mag):
        got = got.cpu().double()
        assert ((got - want).abs() <= want.abs() * 2.0 ** -8 + mag * (2e-7 + 2.0 ** -20) + 1e-30).all()

    if in_place:
        got = flat[off:].reshape(seq, ldi)
        close(got[:, :heads * hd], wq_y, wq_m)
        if kv:
            close(got[:, heads * hd:width], wk_y, wk_m)
        assert torch.equal(got[:, width:].cpu(), x[:, width:])
    else:
        close(bq[:seq, :heads * hd], wq_y, wq_m)
        assert (bq[:seq, heads * hd:] == 7).all() and (bq[seq] == 7).all()
        if not q_only:
            close(bk[:seq, :kv * hd], wk_y, wk_m)
            assert (bk[:seq, kv * hd:] == 7).all() and (bk[seq] == 7).all()
        else:
            assert (bk == 7).all()
        assert torch.equal(flat[off:].reshape(seq, ldi).cpu(), x)     # the inputs stay


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("seq,heads,kv,hd,dims", [(1, 1, 1, 128, (128,)), (3, 5, 1, 128, (32, 48, 48)), (130, 30, 30, 128, (32, 48, 48)),
                                                  (517, 8, 2, 128, (16, 24, 24)), (37, 6, 3, 64, (16, 24, 24)),
                                                  (29, 3, 1, 256, (64, 96, 96)), (6000, 2, 1, 128, (32, 32, 32, 32))])
def test_prologue_vector_kernel(lib, seq, heads, kv, hd, dims, norm, split):
    prologue(lib, seq, heads, kv, hd, dims, split, norm, pad=8)
    prologue(lib, seq, heads, kv, hd, dims, split, norm, in_place=True, pad=16)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("seq,heads,kv,hd,dims,pad,off", [(5, 3, 2, 128, (32, 48, 48), 3, 0), (11, 2, 2, 128, (64, 64), 8, 1),
                                                          (9, 4, 1, 6, (2, 2), 0, 0), (7, 1, 1, 512, (200, 200, 112), 0, 0),
                                                          (13, 5, 5, 96, (32, 32, 32), 0, 0)])
def test_prologue_general_kernel(lib, seq, heads, kv, hd, dims, pad, off, split):
    for norm in (True, False):
        prologue(lib, seq, heads, kv, hd, dims, split, norm, pad=pad, off=off)
    prologue(lib, seq, heads, kv, hd, dims, split, True, in_place=True, pad=pad, off=off)


def test_prologue_queries_only_and_empty(lib):
    prologue(lib, 19, 4, 0, 128, (32, 48, 48), False, True, q_only=True)
    prologue(lib, 19, 4, 2, 128, (32, 48, 48), True, False, q_only=True, pad=8)
    plan = lib.rope_axes((128,), None, 10000.0, False, 128)
    assert lib.iris_b200_qk_norm_rope_axes(None, 128, None, 128, None, None, 256, None, None, None, plan, 0, 1, 1, 128, 1e-6, 0) == 0
    assert lib.iris_b200_rope_axes_tables(None, None, None, plan, 0, 128) == 0
    done(lib)


def test_prologue_agrees_with_the_table_form(lib):
    """The same rows through the tables and the table-driven prologue: within one bf16 step of each other."""
    seq, heads, dims = 301, 6, (32, 48, 48)
    plan = lib.rope_axes(dims, None, 256.0, False, D)
    pos = positions(5, seq, 3, 1000).cuda()
    x = (randn(6, seq, 2 * heads * D) * 1.3).bfloat16().cuda()
    w = (1.0 + 0.2 * randn(7, D)).cuda()
    cos, sin = torch.empty(seq, 64).cuda(), torch.empty(seq, 64).cuda()
    y = x.clone()
    assert lib.iris_b200_rope_axes_tables(ptr(cos), ptr(sin), ptr(pos), plan, seq, D) == 0
    ld = 2 * heads * D
    assert lib.iris_b200_qk_norm_rope(ptr(y), ptr(y, heads * D), ld, ptr(w), ptr(w), ptr(cos), ptr(sin), seq, heads, D, 1e-6, 0) == 0
    assert lib.iris_b200_qk_norm_rope_axes(ptr(x), ld, ptr(x, heads * D), ld, ptr(x), ptr(x, heads * D), ld, ptr(w), ptr(w),
                                           ptr(pos), plan, seq, heads, heads, D, 1e-6, 0) == 0
    done(lib)
    a, b = x.double(), y.double()
    assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 1e-5).all()


# ---------------------------------------------------------------------------
# block means
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("seq,heads,hd,block,pad,off,masked", [
    (1, 1, 128, 64, 0, 0, False), (64, 2, 128, 64, 0, 0, False), (65, 3, 128, 64, 8, 0, True), (1000, 5, 128, 128, 0, 0, True),
    (777, 2, 128, 1, 0, 0, True), (300, 2, 128, 1000, 0, 0, True), (130, 3, 80, 16, 0, 0, True), (97, 3, 7, 10, 5, 0, True),
    (200, 2, 128, 32, 3, 1, False), (4096, 30, 128, 512, 0, 0, False)])
def test_block_means(lib, seq, heads, hd, block, pad, off, masked):
    ld = heads * hd + pad
    x = (randn(seq, seq, ld) + 0.5).bfloat16()
    mask = None
    if masked:
        mask = (torch.rand(seq, generator=torch.Generator().manual_seed(2)) < 0.7).int() * 5 - (torch.arange(seq) % 11 == 0).int()
        if seq > 2 * block:
            mask[block:2 * block] = 0                                   # a block without any row
        x[mask == 0] = NAN                                              # what masked rows hold must not matter
    n = (seq + block - 1) // block
    flat = torch.cat([torch.zeros(off).bfloat16(), x.reshape(-1)]).cuda()
    out, counts, dm = torch.full((n + 1, heads, hd), NAN).cuda(), torch.full((n + 1,), -7, dtype=torch.int32).cuda(), gpu(mask)
    assert lib.iris_b200_block_means(ptr(out), ptr(counts), ptr(flat, off), ld, seq, heads, hd, block, ptr(dm)) == 0
    done(lib)
    want, wc, mag = ref.means(x[:, :heads * hd], heads, hd, block, mask)
    assert torch.equal(counts[:n].cpu(), wc) and counts[n] == -7 and out[n].isnan().all()
    got = out[:n].cpu().double()
    assert ((got - want).abs() <= 2.0 ** -24 * want.abs() + 15 * 2.0 ** -24 * mag).all()
    again = torch.empty(n, heads, hd).cuda()
    assert lib.iris_b200_block_means(ptr(again), None, ptr(flat, off), ld, seq, heads, hd, block, ptr(dm)) == 0
    done(lib)
    assert torch.equal(again, out[:n])


def test_block_means_of_a_growing_cache(lib):
    """The last block alone gives the same values as the whole sequence."""
    heads, block, seq = 4, 64, 300
    x = randn(1, seq, heads * D).bfloat16().cuda()
    n = (seq + block - 1) // block
    whole, last = torch.empty(n, heads, D).cuda(), torch.zeros(n, heads, D).cuda()
    assert lib.iris_b200_block_means(ptr(whole), None, ptr(x), heads * D, seq, heads, D, block, None) == 0
    assert lib.iris_b200_block_means(ptr(last, (n - 1) * heads * D), None, ptr(x, (n - 1) * block * heads * D), heads * D,
                                     seq - (n - 1) * block, heads, D, block, None) == 0
    done(lib)
    assert torch.equal(whole[n - 1], last[n - 1]) and not last[:n - 1].any()


# ---------------------------------------------------------------------------
# lists
# ---------------------------------------------------------------------------

def run_select(lib, qm, km, counts, topk, first, last):
    nq, heads, hd = qm.shape
    nk, kv = km.shape[:2]
    out = torch.full((heads * nq * topk + 1,), -9, dtype=torch.int32).cuda()
    a, b, c = qm.cuda(), km.cuda(), gpu(counts)
    assert lib.iris_b200_block_select(ptr(out), ptr(a), ptr(b), ptr(c), nq, nk, heads, kv, hd, topk, first, last) == 0
    done(lib)
    assert out[-1] == -9
    return out[:-1].reshape(heads, nq, topk).cpu()


@pytest.mark.parametrize("nq,nk,heads,kv,hd,topk,first,last", [
    (1, 1, 1, 1, 128, 1, 0, 0), (1, 5, 2, 1, 128, 9, 1, 1), (9, 33, 6, 3, 128, 7, 2, 0), (5, 264, 3, 3, 128, 40, 8, 3),
    (17, 31, 4, 4, 64, 31, 0, 0), (3, 40, 2, 2, 24, 5, 0, 5), (3, 40, 2, 1, 7, 5, 0, 2), (2, 3500, 2, 2, 128, 64, 1, 2),
    (2, 6000, 5, 1, 16, 100, 0, 0), (1, 23552, 1, 1, 16, 17, 0, 0), (4, 2, 2, 2, 128, 6, 3, 3),
    (1, 130, 4, 4, 128, 30, 0, 0), (1, 515, 8, 2, 128, 64, 1, 2), (2, 1030, 16, 2, 128, 1, 0, 0), (3, 23552, 1, 1, 24, 300, 0, 1),
    (1, 600, 5, 1, 128, 599, 0, 0), (21, 300, 3, 1, 512, 20, 0, 0)])
def test_block_select(lib, nq, nk, heads, kv, hd, topk, first, last):
    qm, km = randn(nk, nq, heads, hd), randn(nk + 1, nk, kv, hd)
    gen = torch.Generator().manual_seed(nq)
    for counts in (None, torch.randint(0, 3, (nk,), generator=gen, dtype=torch.int32), torch.zeros(nk, dtype=torch.int32)):
        if nk > 4000 and counts is not None:
            continue
        got = run_select(lib, qm, km, counts, topk, first, last)
        assert torch.equal(got, ref.select(qm, km, counts, topk, first, last))


def test_block_select_ties_go_to_the_lowest_block(lib):
    """Integers, so that every score is exact and most are equal; both zeros; values that only 64 bits tell apart."""
    gen = torch.Generator().manual_seed(3)
    qm = torch.randint(-1, 2, (6, 2, 32), generator=gen).float()
    km = torch.randint(-1, 2, (70, 2, 32), generator=gen).float()
    qm[0] = 0.0
    km[::2] *= -1.0
    assert torch.equal(run_select(lib, qm, km, None, 11, 1, 1), ref.select(qm, km, None, 11, 1, 1))
    same = torch.ones(40, 1, 128)
    same[7, 0, 0] = 1.0 + 2.0 ** -23
    one = torch.ones(1, 1, 128)
    one[0, 0, 0] = 1.0 + 2.0 ** -20
    want = torch.tensor([[[0, 1, 7]]], dtype=torch.int32)
    assert torch.equal(run_select(lib, one, same, None, 3, 0, 0), want)


@pytest.mark.parametrize("nq,nk,kv", [(16, 100, 150), (16, 264, 150), (16, 500, 150), (16, 700, 150), (5, 300, 150), (2, 500, 150),
                                      (1, 1100, 150), (2, 2000, 1), (1, 23552, 1), (16, 600, 1)])
def test_block_select_many_equal_scores(lib, nq, nk, kv):
    """Scores that are whole numbers between -8 and 8, so that hundreds of blocks are equal at the cut, over the sizes that
    share a row between one, two, four and eight warps in one to eight CTAs."""
    gen = torch.Generator().manual_seed(nk)
    qm, km = torch.zeros(nq, kv, 128), torch.zeros(nk, kv, 128)
    qm[..., ::16] = torch.randint(-1, 2, (nq, kv, 8), generator=gen).float()
    km[..., ::16] = torch.randint(-1, 2, (nk, kv, 8), generator=gen).float()
    counts = (torch.rand(nk, generator=gen) < 0.9).int()
    first, last = 2, 3
    score = torch.einsum("qhd,khd->hqk", qm.double(), km.double())
    j = torch.arange(nk)
    rank = score * nk - j                    # higher first, equal ones by the lowest block
    rank = torch.where(((j < first) | (j >= nk - last)) & (counts > 0), rank + 100.0 * nk, rank)
    rank = torch.where(counts > 0, rank, torch.full_like(rank, -100.0 * nk))
    for topk in (5, nk // 3, nk - 1):
        n = min(topk, int(counts.sum()))
        want = torch.full((kv, nq, topk), -1, dtype=torch.int32)
        want[..., :n] = rank.topk(n, dim=-1)[1].sort(-1)[0].int()
        assert torch.equal(run_select(lib, qm, km, counts, topk, first, last), want)


def test_block_select_unaligned_means(lib):
    """Means at an odd word: the same lists."""
    nq, nk, heads, kv = 5, 300, 4, 2
    qm, km = randn(1, nq, heads, D), randn(2, nk, kv, D)
    a, b = torch.zeros(qm.numel() + 1).cuda(), torch.zeros(km.numel() + 1).cuda()
    a[1:], b[1:] = qm.flatten(), km.flatten()
    out = torch.zeros(heads, nq, 20, dtype=torch.int32).cuda()
    assert lib.iris_b200_block_select(ptr(out), ptr(a, 1), ptr(b, 1), None, nq, nk, heads, kv, D, 20, 1, 1) == 0
    done(lib)
    assert torch.equal(out.cpu(), ref.select(qm, km, None, 20, 1, 1))


def test_block_select_values_that_are_not_finite(lib):
    qm, km = randn(1, 2, 1, 128), randn(2, 20, 1, 128)
    km[4] = NAN                              # ranks last, but before nothing
    km[9, 0, 0] = float("inf")
    qm[0, 0, 0], qm[1, 0, 0] = 2.0, -2.0     # block 9 scores +inf for the first row, -inf for the second
    for topk in (1, 5, 18, 19, 20):
        assert torch.equal(run_select(lib, qm, km, None, topk, 0, 0), ref.select(qm, km, None, topk, 0, 0))


def test_block_select_without_blocks(lib):
    qm = randn(1, 3, 2, 128).cuda()
    out = torch.zeros(2, 3, 4, dtype=torch.int32).cuda()
    assert lib.iris_b200_block_select(ptr(out), ptr(qm), None, None, 3, 0, 2, 2, 128, 4, 0, 0) == 0
    done(lib)
    assert (out == -1).all()


# ---------------------------------------------------------------------------
# attention over the lists
# ---------------------------------------------------------------------------

def random_lists(seed, heads, nq, nk, n, junk=False):
    gen = torch.Generator().manual_seed(seed)
    out = torch.full((heads, nq, n), -1, dtype=torch.int32)
    for h in range(heads):
        for i in range(nq):
            m = min(n, nk)
            if junk:
                m = int(torch.randint(0, m + 1, (1,), generator=gen))
            pick = torch.randperm(nk, generator=gen)[:m].sort()[0].int()
            out[h, i, :m] = pick
            if junk:                         # gaps, blocks that do not exist, any order
                out[h, i, m:] = torch.tensor([-1, nk, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)[
                    torch.randint(0, 4, (n - m,), generator=gen)]
                out[h, i] = out[h, i][torch.randperm(n, generator=gen)]
    return out


def run_attention(lib, q, k, v, heads, kv, hd, mask, lists, q_block, k_block, kernel, pad=0, scale=None):
    """q / k / v float tensors [rows, heads * hd]; out with guard columns and a guard row."""
    scale = scale or hd ** -0.5
    sq, sk = q.shape[0], k.shape[0]
    fused = torch.full((max(sk, 1), 2 * kv * hd + pad), NAN).bfloat16()
    fused[:sk, :kv * hd], fused[:sk, kv * hd:2 * kv * hd] = k, v
    dq = torch.full((max(sq, 1), heads * hd + pad), NAN).bfloat16()
    dq[:sq, :heads * hd] = q
    out = torch.full((sq + 1, heads * hd + pad), 7.0).bfloat16().cuda()
    dq, df, dl, dm = dq.cuda(), fused.cuda(), lists.cuda(), gpu(mask)
    rc = lib.iris_b200_attention_blocks(ptr(out), heads * hd + pad, ptr(dq), heads * hd + pad, ptr(df), 2 * kv * hd + pad,
                                        ptr(df, kv * hd), 2 * kv * hd + pad, sq, sk, heads, kv, hd, scale, ptr(dm), ptr(dl), lists.shape[2],
                                        q_block, k_block, kernel)
    assert rc == 0, rc
    done(lib)
    assert (out[sq] == 7).all() and (out[:, heads * hd:] == 7).all()
    return out[:sq, :heads * hd].cpu().double()


def check_attention(lib, sq, sk, heads, kv, hd, n, q_block, k_block, kernel, masked=False, pad=0, junk=False, seed=0, scale=None,
                    gain=1.0):
    nq, nk = -(-sq // q_block), -(-sk // k_block)
    q, k, v = ((gain if i < 2 else 1.0) * randn(seed + i, r, c) for i, (r, c) in
               enumerate([(sq, heads * hd), (sk, kv * hd), (sk, kv * hd)]))
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    mask = None
    if masked:
        mask = (torch.rand(sk, generator=torch.Generator().manual_seed(seed + 9)) < 0.8).int() * 3
        mask[sk - sk // 8:] = 0
        k[mask == 0], v[mask == 0] = NAN, NAN
        v[(mask == 0) & (torch.arange(sk) % 2 == 0)] = float("inf")
    lists = random_lists(seed, heads, nq, nk, n, junk)
    got = run_attention(lib, q, k, v, heads, kv, hd, mask, lists, q_block, k_block, kernel, pad, scale)
    want, mag = ref.attention(q, k, v, heads, kv, hd, scale or hd ** -0.5, mask, lists, q_block, k_block)
    assert got.isfinite().all()
    worst = ((got - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mag + 1e-30)).max().item()
    assert worst <= 0.0, worst
    return got


GENERAL = [  # sq, sk, heads, kv, hd, list_len, q_block, k_block, masked, pad, junk
    (1, 1, 1, 1, 128, 1, 1, 1, False, 0, False), (37, 53, 3, 1, 128, 3, 5, 7, True, 0, True), (40, 64, 2, 2, 64, 4, 16, 16, False, 0, False),
    (9, 200, 4, 2, 80, 2, 9, 64, True, 3, True), (20, 30, 2, 2, 7, 3, 8, 4, False, 0, False), (11, 70, 1, 1, 512, 2, 4, 33, True, 0, False),
    (130, 130, 2, 2, 128, 3, 128, 48, True, 1, True)]


@pytest.mark.parametrize("sq,sk,heads,kv,hd,n,qb,kb,masked,pad,junk", GENERAL)
def test_attention_general_kernel(lib, sq, sk, heads, kv, hd, n, qb, kb, masked, pad, junk):
    check_attention(lib, sq, sk, heads, kv, hd, n, qb, kb, GENERIC, masked, pad, junk)
    check_attention(lib, sq, sk, heads, kv, hd, n, qb, kb, AUTO, masked, pad, junk, seed=5)


TENSOR = [  # sq, sk, heads, kv, list_len, q_block, k_block, masked, pad, junk
    (1, 1, 1, 1, 1, 1, 64, False, 0, False), (128, 128, 1, 1, 1, 128, 128, False, 0, False), (128, 128, 2, 2, 2, 128, 64, False, 8, False),
    (129, 200, 2, 1, 3, 128, 64, True, 0, False), (300, 333, 3, 3, 4, 128, 64, True, 16, True), (300, 333, 3, 3, 20, 128, 16, True, 0, True),
    (517, 517, 2, 2, 9, 256, 32, True, 0, True), (260, 900, 4, 2, 2, 384, 256, True, 0, True), (64, 700, 2, 2, 3, 100, 128, True, 0, False),
    (77, 2000, 2, 2, 2, 16, 512, True, 0, False), (3, 4096, 4, 1, 64, 1, 64, True, 0, True), (2, 8192, 2, 1, 32, 2, 256, False, 0, False),
    (1, 4096, 8, 2, 40, 1, 64, False, 0, False), (40, 3000, 2, 2, 47, 40, 64, True, 0, True), (128, 3000, 1, 1, 33, 128, 64, True, 0, True)]


@pytest.mark.parametrize("sq,sk,heads,kv,n,qb,kb,masked,pad,junk", TENSOR)
def test_attention_tensor_kernel(lib, sq, sk, heads, kv, n, qb, kb, masked, pad, junk):
    check_attention(lib, sq, sk, heads, kv, 128, n, qb, kb, TCGEN05, masked, pad, junk)
    check_attention(lib, sq, sk, heads, kv, 128, n, qb, kb, TCGEN05, masked, pad, junk, seed=7, gain=3.0)


ROWS = [  # sq, sk, heads, kv, hd, list_len, k_block, masked, pad, junk
    (1, 1, 1, 1, 128, 1, 1, False, 0, False), (1, 9, 2, 1, 64, 3, 7, False, 0, True), (5, 333, 3, 3, 256, 9, 16, True, 8, True),
    (3, 4096, 4, 1, 128, 64, 64, True, 0, True), (1, 4096, 8, 2, 128, 40, 64, False, 0, False), (1, 2000, 2, 2, 64, 2, 900, True, 0, False),
    (40, 700, 12, 4, 128, 5, 48, True, 16, True), (2, 9000, 1, 1, 256, 33, 33, True, 0, False), (1, 5000, 1, 1, 128, 300, 16, True, 0, True),
    (300, 1000, 2, 2, 64, 17, 32, True, 0, True)]


@pytest.mark.parametrize("sq,sk,heads,kv,hd,n,kb,masked,pad,junk", ROWS)
def test_attention_row_kernel(lib, sq, sk, heads, kv, hd, n, kb, masked, pad, junk):
    check_attention(lib, sq, sk, heads, kv, hd, n, 1, kb, AUTO, masked, pad, junk)
    check_attention(lib, sq, sk, heads, kv, hd, n, 1, kb, AUTO, masked, pad, junk, seed=7, gain=3.0)
    if sq == 1:                              # the only query, whatever its block is called
        check_attention(lib, sq, sk, heads, kv, hd, n, 100, kb, AUTO, masked, pad, junk)


def test_attention_row_kernel_without_keys_and_not_finite(lib):
    q, k, v = (randn(i, r, 256).bfloat16() for i, r in enumerate((4, 200, 200)))
    mask = torch.ones(200, dtype=torch.int32)
    mask[64:128] = 0                          # block 1 is masked as a whole
    v[70:90], k[100] = NAN, NAN               # and holds no numbers
    v[10, 5], k[140] = NAN, NAN               # seen by the lists that hold blocks 0 and 2
    lists = torch.tensor([[[-1, -1, -1], [9, -5, 4], [1, -1, 1], [3, -1, 1]], [[0, 3, 1], [2, 2, -1], [3, 3, 9], [1, 9, 3]]], dtype=torch.int32)
    got = run_attention(lib, q, k, v, 2, 2, 128, mask, lists, 1, 64, AUTO)
    bad = got.isnan()
    assert (got[:3, :128] == 0).all() and not bad[3].any() and not bad[2].any()
    assert not bad[0, 128:].any() and bad[1, 128:].all()         # column 5 of row 10 is head 0's
    got = run_attention(lib, q, k, v, 2, 2, 128, mask, lists.flip(0), 1, 64, AUTO)
    assert got[0, :128].isnan().sum() == 1 and got[0, 5].isnan()
    want, _ = ref.attention(q[2:], k[:140], v[:140], 2, 2, 128, 128 ** -0.5, mask[:140], torch.full((2, 2, 1), 0), 1, 8)
    got = run_attention(lib, q[2:], k[:140], v[:140], 2, 2, 128, mask[:140], torch.full((2, 2, 1), 0, dtype=torch.int32), 1, 8, AUTO)
    assert (got - want).abs().max() < 0.05
    for sk, n in ((0, 2), (200, 0)):
        got = run_attention(lib, q, k[:sk], v[:sk], 2, 2, 128, None, torch.zeros(2, 4, n, dtype=torch.int32), 1, 64, AUTO)
        assert (got == 0).all()


@pytest.mark.parametrize("sq,heads,n,qb,masked,junk", [(2500, 30, 3, 128, False, False), (3700, 12, 35, 200, True, True),
                                                       (11, 64, 5, 1, True, False)])
def test_attention_tensor_kernel_more_tiles_than_fit_at_once(lib, sq, heads, n, qb, masked, junk):
    check_attention(lib, sq, 2900, heads, 2, 128, n, qb, 64, TCGEN05, masked, 0, junk)


@pytest.mark.parametrize("kb,n", [(16, 11), (32, 6), (64, 3), (128, 2), (256, 2)])
def test_attention_tensor_kernel_tiles_without_keys_among_others(lib, kb, n):
    """Empty lists and lists of masked blocks only, in runs, between tiles with keys, several tiles to a CTA."""
    sq, sk, heads = 3900, 2100, 20
    nq, nk = -(-sq // 128), -(-sk // kb)
    gen = torch.Generator().manual_seed(kb)
    q, k, v = (randn(kb + i, r, D if i else heads * D).bfloat16() for i, r in enumerate((sq, sk, sk)))
    mask = (torch.rand(sk, generator=gen) < 0.97).int()
    mask[512:1024] = 0                       # whole blocks of every size
    k[mask == 0], v[mask == 0] = NAN, NAN
    lists = random_lists(kb + 7, heads, nq, nk, n)
    what = torch.randint(0, 4, (heads, nq), generator=gen)
    masked = torch.arange(512 // kb, 1024 // kb)
    for h in range(heads):
        for i in range(nq):
            if what[h, i] == 0:
                lists[h, i] = -1
            elif what[h, i] == 1:
                lists[h, i] = masked[torch.randint(0, len(masked), (n,), generator=gen)].int()
    got = run_attention(lib, q, k, v, heads, 1, D, mask, lists, 128, kb, TCGEN05)
    want, mag = ref.attention(q, k, v, heads, 1, D, D ** -0.5, mask, lists, 128, kb)
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mag).all()
    for h in range(heads):
        for i in range(nq):
            if what[h, i] < 2:
                assert (got[i * 128:(i + 1) * 128, h * D:(h + 1) * D] == 0).all()


@pytest.mark.parametrize("sq,heads,n", [(1, 8, 40), (300, 3, 6), (100, 2, 40)])
def test_attention_tensor_kernel_growing_scores(lib, sq, heads, n):
    """Scores that rise from block to block, so that the running maximum moves and O is rescaled."""
    sk, kb = 2560, 64
    q = torch.ones(sq, heads * 128) + 0.1 * randn(1, sq, heads * 128)
    k = (torch.arange(sk).reshape(sk, 1) // kb * 0.02 - 0.3) + 0.05 * randn(2, sk, heads * 128)
    v = randn(3, sk, heads * 128)
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    lists = random_lists(4, heads, -(-sq // 128), sk // kb, n)
    got = run_attention(lib, q, k, v, heads, heads, 128, None, lists, 128, kb, TCGEN05, scale=0.5)
    want, mag = ref.attention(q, k, v, heads, heads, 128, 0.5, None, lists, 128, kb)
    # |s| up to 64 * 0.5 = 32 here: a dot product of magnitude 64 off by 2^-17 relative, 2^-10 in s
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * mag).all()


def test_attention_values_that_are_not_finite_show(lib):
    """A NaN in a key or value row that counts reaches the rows that see it, and no others."""
    q, k, v = (randn(i, 256, 128).bfloat16() for i in range(3))
    v[70, 5] = NAN
    k[200] = NAN
    lists = torch.tensor([[[0, 1], [2, 3]]], dtype=torch.int32)
    for kernel in (GENERIC, TCGEN05):
        got = run_attention(lib, q, k, v, 1, 1, 128, None, lists, 128, 64, kernel)
        bad = got.isnan()
        assert bad[:128, 5].all() and bad[:128].sum() == 128 and bad[128:].all()


@pytest.mark.parametrize("kernel", [GENERIC, AUTO])
def test_attention_rows_without_keys(lib, kernel):
    q, k, v = (randn(i, r, 256).bfloat16() for i, r in enumerate((300, 200, 200)))
    lists = random_lists(1, 2, 3, 4, 3)
    lists[0, 1] = -1                          # an empty list
    lists[1, 2] = torch.tensor([9, -5, 4])    # none of its blocks exists
    mask = torch.ones(200, dtype=torch.int32)
    mask[64:128] = 0                          # block 1 is masked as a whole
    lists[1, 0] = torch.tensor([1, -1, -1])
    got = run_attention(lib, q, k, v, 2, 2, 128, mask, lists, 128, 64, kernel)
    want, _ = ref.attention(q, k, v, 2, 2, 128, 128 ** -0.5, mask, lists, 128, 64)
    for h, rows in ((0, slice(128, 256)), (1, slice(256, 300)), (1, slice(0, 128))):
        assert (got[rows, h * 128:(h + 1) * 128] == 0).all()
    assert (got - want).abs().max() < 0.1
    # no keys at all, and lists of no length
    for sk, n in ((0, 2), (200, 0)):
        got = run_attention(lib, q, k[:sk], v[:sk], 2, 2, 128, None, torch.zeros(2, 3, n, dtype=torch.int32), 128, 64, kernel)
        assert (got == 0).all()


@pytest.mark.parametrize("kernel", [GENERIC, AUTO])
def test_attention_block_listed_twice_counts_twice(lib, kernel):
    q, k, v = (randn(20 + i, r, 128).bfloat16() for i, r in enumerate((50, 256, 256)))
    lists = torch.tensor([[[1, 3, 1, -1]]], dtype=torch.int32)
    for rows in (50, 1):
        got = run_attention(lib, q[:rows], k, v, 1, 1, 128, None, lists, 50, 64, kernel)
        want, mag = ref.attention(q[:rows], k, v, 1, 1, 128, 128 ** -0.5, None, lists, 50, 64)
        assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mag).all()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def test_the_operators_together(lib):
    """Positions -> norm and rotation -> means -> lists -> attention, as a block of a model runs them; with lists that hold
    every block the result is that of the dense attention."""
    heads, kv, seq, qb, kb, dims = 4, 2, 1000, 128, 64, (32, 48, 48)
    plan = lib.rope_axes(dims, (1.0, 1.0, 1.0), 256.0, False, D)
    pos = torch.stack([torch.arange(seq) // 100, torch.arange(seq) // 10 % 10, torch.arange(seq) % 10], 1).int().cuda()
    ld = (heads + 2 * kv) * D
    x = (randn(1, seq, ld) * 1.4).bfloat16().cuda()
    w = (1.0 + 0.2 * randn(2, D)).cuda()
    mask = torch.ones(seq, dtype=torch.int32)
    mask[950:] = 0
    dm = mask.cuda()
    nq, nk = -(-seq // qb), -(-seq // kb)
    q, k = torch.empty(seq, heads * D).bfloat16().cuda(), torch.empty(seq, kv * D).bfloat16().cuda()
    qm, km = torch.empty(nq, heads, D).cuda(), torch.empty(nk, kv, D).cuda()
    counts = torch.empty(nk, dtype=torch.int32).cuda()
    v = x[:, (heads + kv) * D:].contiguous()

    def run(topk):
        lists = torch.empty(heads, nq, topk, dtype=torch.int32).cuda()
        out = torch.empty(seq, heads * D).bfloat16().cuda()
        rc = lib.iris_b200_qk_norm_rope_axes(ptr(q), heads * D, ptr(k), kv * D, ptr(x), ptr(x, heads * D), ld, ptr(w), ptr(w),
                                             ptr(pos), plan, seq, heads, kv, D, 1e-5, 0)
        rc |= lib.iris_b200_block_means(ptr(qm), None, ptr(q), heads * D, seq, heads, D, qb, None)
        rc |= lib.iris_b200_block_means(ptr(km), ptr(counts), ptr(k), kv * D, seq, kv, D, kb, ptr(dm))
        rc |= lib.iris_b200_block_select(ptr(lists), ptr(qm), ptr(km), ptr(counts), nq, nk, heads, kv, D, topk, 1, 1)
        rc |= lib.iris_b200_attention_blocks(ptr(out), heads * D, ptr(q), heads * D, ptr(k), kv * D, ptr(v), kv * D, seq, seq,
                                             heads, kv, D,
                                             D ** -0.5, ptr(dm), ptr(lists), topk, qb, kb, AUTO)
        assert rc == 0
        done(lib)
        return lists.cpu(), out.cpu()

    lists, out = run(6)
    xc, wc = x.cpu(), w.cpu()
    ang = ref.angles(pos.cpu(), dims, None, 256.0, False, D)
    wq, _ = ref.norm_rope(xc[:, :heads * D], heads, D, wc, 1e-5, ang, False)
    assert ((q.cpu().double() - wq).abs() <= 2.0 ** -8 * wq.abs() + 1e-5).all()
    # from here on against the rounded rows that the attention reads
    rq, _, _ = ref.means(q.cpu(), heads, D, qb)
    rk, rc, _ = ref.means(k.cpu(), kv, D, kb, mask)
    assert torch.equal(counts.cpu(), rc)
    assert torch.equal(lists, ref.select(qm.cpu(), km.cpu(), rc, 6, 1, 1))
    assert (qm.cpu().double() - rq).abs().max() < 1e-6 and (km.cpu().double() - rk).abs().max() < 1e-6
    want, mag = ref.attention(q.cpu(), k.cpu(), v.cpu(), heads, kv, D, D ** -0.5, mask, lists, qb, kb)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mag).all()

    lists, out = run(nk)                     # every block with a valid row
    dense = torch.empty(seq, heads * D).bfloat16().cuda()
    kk = k.reshape(seq, kv, D).repeat_interleave(heads // kv, 1).reshape(seq, heads * D).contiguous()
    vv = v.reshape(seq, kv, D).repeat_interleave(heads // kv, 1).reshape(seq, heads * D).contiguous()
    assert lib.iris_b200_attention_ex(ptr(dense), heads * D, ptr(q), ptr(kk), ptr(vv), heads * D, seq, seq, heads, heads, D,
                                      D ** -0.5, 0, ptr(dm), 0) == 0
    done(lib)
    a, b = out.double(), dense.cpu().double()
    mag = ref.attention(q.cpu(), k.cpu(), v.cpu(), heads, kv, D, D ** -0.5, mask, lists, qb, kb)[1]
    assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + (2.0 ** -7 + 2.0 ** -11) * mag).all()


@pytest.mark.parametrize("kernel", [GENERIC, TCGEN05, AUTO])
@pytest.mark.parametrize("sq", [1, 100])
def test_attention_blocks_larger_than_the_sequences(lib, kernel, sq):
    """One block holds all keys, one all queries: the dense attention."""
    check_attention(lib, sq, 300, 2, 1, 128, 1, 2 ** 31 - 1, 2 ** 30, kernel)
    check_attention(lib, sq, 300, 2, 1, 128, 3, 2 ** 30, 2 ** 31 - 128, kernel, masked=True)


FIRST_CALLS = """
import sys, torch
sys.path[:0] = [%r, %r]
import __graft_entry__ as ge
lib = ge.load_package().load()
lib.init()
s = torch.cuda.Stream()
D, seq, heads = 128, 1000, 2
x = torch.randn(seq, 3 * heads * D, device="cuda").bfloat16()
q, k, out = (torch.zeros(seq, heads * D, device="cuda").bfloat16() for _ in range(3))
pos = torch.randint(0, 90, (seq, 3), dtype=torch.int32, device="cuda")
cos, sin = torch.zeros(seq, 64, device="cuda"), torch.zeros(seq, 64, device="cuda")
qm, km = torch.zeros(8, heads, D, device="cuda"), torch.zeros(16, heads, D, device="cuda")
lists = torch.zeros(heads, 8, 5, dtype=torch.int32, device="cuda")
plan = lib.rope_axes((32, 48, 48), None, 256.0, False, D)
p = lambda t: t.data_ptr()
torch.cuda.synchronize()

def run():
    ld, w = 3 * heads * D, heads * D
    assert lib.iris_b200_use_stream(torch.cuda.current_stream().cuda_stream) == 0
    rc = lib.iris_b200_rope_axes_tables(p(cos), p(sin), p(pos), plan, seq, D)
    rc |= lib.iris_b200_qk_norm_rope_axes(p(q), w, p(k), w, p(x), p(x) + 2 * w, ld, None, None, p(pos), plan, seq, heads, heads, D, 0.0, 0)
    rc |= lib.iris_b200_block_means(p(qm), None, p(q), w, seq, heads, D, 128, None)
    rc |= lib.iris_b200_block_means(p(km), None, p(k), w, seq, heads, D, 64, None)
    rc |= lib.iris_b200_block_select(p(lists), p(qm), p(km), None, 8, 16, heads, heads, D, 5, 0, 0)
    rc |= lib.iris_b200_attention_blocks(p(out), w, p(q), w, p(k), w, p(x) + 4 * w, ld, seq, seq, heads, heads, D, 0.1, None, p(lists), 5,
                                         128, 64, 0)
    rc |= lib.iris_b200_attention_blocks(p(out), w, p(q), w, p(k), w, p(x) + 4 * w, ld, 1, seq, heads, heads, D, 0.1, None, p(lists), 5,
                                         1, 64, 0)
    assert rc == 0, lib.iris_b200_last_error()

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    run()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (cos, sin, q, k, qm, km, lists, out)]
with torch.cuda.stream(s):
    run()
torch.cuda.synchronize()
assert got[7].abs().sum() > 0
assert all(torch.equal(a, b) for a, b in zip(got, (cos, sin, q, k, qm, km, lists, out)))
lib.check()
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing that a first call sets up is closed to a capture."""
    here = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS % (os.path.dirname(here), here)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


def test_offsets_that_pass_32_bits(lib):
    """Rows a long way apart: the last ones lie behind 2^31 elements of their tensor."""
    seq, ld = 262400, 8320
    x = torch.empty(seq, ld, dtype=torch.bfloat16, device="cuda")
    rows = randn(1, seq, D).bfloat16().cuda()
    x[:, :D] = rows
    assert seq * ld > 2 ** 31 + 2 ** 25
    means = torch.empty(seq // 64, D).cuda()
    assert lib.iris_b200_block_means(ptr(means), None, ptr(x), ld, seq, 1, D, 64, None) == 0
    done(lib)
    assert (means.double() - rows.double().reshape(-1, 64, D).mean(1)).abs().max() < 1e-6
    lists = torch.tensor([[[0, seq // 64 - 1, seq // 128]]], dtype=torch.int32)
    keys = torch.cat([torch.arange(b * 64, b * 64 + 64) for b in lists[0, 0].tolist()])
    q, kr = randn(2, 100, D).bfloat16(), rows[keys.cuda()].cpu()
    want, mag = ref.attention(q, kr, kr, 1, 1, D, D ** -0.5, None, torch.tensor([[[0, 1, 2]]]), 100, 64)
    dq, dl = q.cuda(), lists.cuda()
    for kernel in (GENERIC, TCGEN05):
        out = torch.zeros(100, D).bfloat16().cuda()
        assert lib.iris_b200_attention_blocks(ptr(out), D, ptr(dq), D, ptr(x), ld, ptr(x), ld, 100, seq, 1, 1, D, D ** -0.5, None,
                                              ptr(dl), 3, 100, 64, kernel) == 0
        done(lib)
        got = out.cpu().double()
        assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mag).all()
    plan = lib.rope_axes((128,), None, 256.0, False, D)
    pos = torch.zeros(seq, 1, dtype=torch.int32).cuda()        # no turn: rows come back as they are
    x[:, D] = 0.0
    for offset in (0, 1):                    # 16-byte kernel, general kernel
        rows = x[:, offset:offset + D].clone()
        assert lib.iris_b200_qk_norm_rope_axes(ptr(x, offset), ld, None, 0, ptr(x, offset), None, ld, None, None, ptr(pos), plan, seq, 1,
                                               0, D, 0.0, 0) == 0
        done(lib)
        if offset == 0:
            assert torch.equal(x[:, :D], rows)
        else:
            assert torch.equal(x[:, 1:D], rows[:, :-1])


def test_calls_behind_one_another_see_what_the_last_one_wrote(lib):
    """The launches overlap at their ends and reuse the same buffers: each has to read what the call before it wrote, not what
    it may have read there one call earlier."""
    heads, seq, qb, kb, topk = 8, 2048, 128, 64, 6
    nq, nk = seq // qb, seq // kb
    xs = [(randn(s, seq, heads * D) * (1.0 + s)).bfloat16().cuda() for s in range(3)]
    poss = [positions(s, seq, 3, 900).cuda() for s in range(3)]
    plan = lib.rope_axes((32, 48, 48), None, 256.0, False, D)
    q, pos = torch.zeros(seq, heads * D).bfloat16().cuda(), torch.zeros(seq, 3, dtype=torch.int32).cuda()
    qm, km = torch.zeros(nq, heads, D).cuda(), torch.zeros(nk, heads, D).cuda()
    lists = torch.zeros(heads, nq, topk, dtype=torch.int32).cuda()

    def step(i, out, kept, cos, sin):
        pos.copy_(poss[i])
        rc = lib.iris_b200_rope_axes_tables(ptr(cos), ptr(sin), ptr(pos), plan, seq, D)
        rc |= lib.iris_b200_qk_norm_rope_axes(ptr(q), heads * D, None, 0, ptr(xs[i]), None, heads * D, None, None, ptr(pos), plan,
                                              seq, heads, 0, D, 1e-6, 0)
        rc |= lib.iris_b200_block_means(ptr(qm), None, ptr(q), heads * D, seq, heads, D, qb, None)
        rc |= lib.iris_b200_block_means(ptr(km), None, ptr(q), heads * D, seq, heads, D, kb, None)
        rc |= lib.iris_b200_block_select(ptr(lists), ptr(qm), ptr(km), None, nq, nk, heads, heads, D, topk, 0, 0)
        rc |= lib.iris_b200_attention_blocks(ptr(out), heads * D, ptr(q), heads * D, ptr(q), heads * D, ptr(xs[i]), heads * D, seq, seq,
                                             heads, heads, D, D ** -0.5, None, ptr(lists), topk, qb, kb, AUTO)
        rc |= lib.iris_b200_block_select(ptr(kept), ptr(qm), ptr(km), None, nq, nk, heads, heads, D, topk, 0, 0)
        assert rc == 0

    def buffers():
        return (torch.zeros(seq, heads * D).bfloat16().cuda(), torch.zeros_like(lists), torch.zeros(seq, D // 2).cuda(),
                torch.zeros(seq, D // 2).cuda())

    alone = []
    for i in range(3):
        alone.append(buffers())
        step(i, *alone[i])
        done(lib)
    runs = [buffers() for _ in range(30)]
    for n, b in enumerate(runs):
        step(n % 3, *b)
    done(lib)
    for n, b in enumerate(runs):
        assert all(torch.equal(x, y) for x, y in zip(b, alone[n % 3])), n


def test_large_calls_on_several_streams_at_once(lib):
    """Two attentions over key blocks that each fill the device, single rows, lists and the dense attention side by side: what
    they give alone."""
    heads, seq, qb, kb, n = 16, 4000, 128, 64, 9
    nq, nk = -(-seq // qb), -(-seq // kb)
    home, side = torch.cuda.current_stream(), [torch.cuda.Stream() for _ in range(4)]

    def inputs(seed):
        q, k, v = (randn(seed + i, seq, heads * D).bfloat16().cuda() for i in range(3))
        qm, km = torch.zeros(nq, heads, D).cuda(), torch.zeros(nk, heads, D).cuda()
        return q, k, v, qm, km, torch.zeros(heads, nq, n, dtype=torch.int32).cuda(), torch.zeros_like(q)

    def blocks(x):
        q, k, v, qm, km, lists, out = x
        w = heads * D
        rc = lib.iris_b200_block_means(ptr(qm), None, ptr(q), w, seq, heads, D, qb, None)
        rc |= lib.iris_b200_block_means(ptr(km), None, ptr(k), w, seq, heads, D, kb, None)
        rc |= lib.iris_b200_block_select(ptr(lists), ptr(qm), ptr(km), None, nq, nk, heads, heads, D, n, 1, 0)
        rc |= lib.iris_b200_attention_blocks(ptr(out), w, ptr(q), w, ptr(k), w, ptr(v), w, seq, seq, heads, heads, D, D ** -0.5, None,
                                             ptr(lists), n, qb, kb, TCGEN05)
        return rc

    def rows(x):
        q, k, v, qm, km, lists, out = x
        w = heads * D
        rc = lib.iris_b200_block_means(ptr(km), None, ptr(k), w, seq, heads, D, kb, None)
        rc |= lib.iris_b200_block_select(ptr(lists), ptr(qm), ptr(km), None, 1, nk, heads, heads, D, n, 0, 0)
        rc |= lib.iris_b200_attention_blocks(ptr(out), w, ptr(q), w, ptr(k), w, ptr(v), w, 1, seq, heads, heads, D, D ** -0.5, None,
                                             ptr(lists), n, 1, kb, AUTO)
        return rc

    def dense(x):
        q, k, v, _, _, _, out = x
        w = heads * D
        return lib.iris_b200_attention_ex(ptr(out), w, ptr(q), ptr(k), ptr(v), w, seq, seq, heads, heads, D, D ** -0.5, 0, None, 0)

    work = list(zip((blocks, blocks, rows, dense), (inputs(10 * i) for i in range(4)), side))
    torch.cuda.synchronize()
    alone = []
    for fn, x, _ in work:
        assert fn(x) == 0
        done(lib)
        alone.append((x[5].clone(), x[6].clone()))
        x[6].zero_()
    torch.cuda.synchronize()
    try:
        for _ in range(12):
            for fn, x, s in work:
                assert lib.iris_b200_use_stream(s.cuda_stream) == 0
                assert fn(x) == 0
        torch.cuda.synchronize()
    finally:
        lib.iris_b200_use_stream(home.cuda_stream)
    done(lib)
    for (_, x, _), (lists, out) in zip(work, alone):
        assert torch.equal(x[5], lists) and torch.equal(x[6], out)


def test_captured_and_replayed(lib):
    """A captured run of the chain gives on replay, with new inputs, what eager calls give; two graphs replayed on two streams
    at once do not disturb one another."""
    heads, seq, qb, kb, topk = 2, 384, 128, 64, 3
    nq, nk = 3, 6
    plan = lib.rope_axes((32, 48, 48), None, 256.0, False, D)
    pos = torch.randint(0, 50, (seq, 3), dtype=torch.int32).cuda()

    class Run:
        def __init__(self, seed):
            self.x = randn(seed, seq, 3 * heads * D).bfloat16().cuda()
            self.q, self.k = (torch.zeros(seq, heads * D).bfloat16().cuda() for _ in "qk")
            self.qm, self.km = torch.zeros(nq, heads, D).cuda(), torch.zeros(nk, heads, D).cuda()
            self.lists = torch.zeros(heads, nq, topk, dtype=torch.int32).cuda()
            self.out = torch.zeros(seq, heads * D).bfloat16().cuda()

        def __call__(self):
            lib.iris_b200_use_stream(torch.cuda.current_stream().cuda_stream)
            ld = 3 * heads * D
            rc = lib.iris_b200_qk_norm_rope_axes(ptr(self.q), heads * D, ptr(self.k), heads * D, ptr(self.x), ptr(self.x, heads * D),
                                                 ld, None, None, ptr(pos), plan, seq, heads, heads, D, 1e-6, 1)
            rc |= lib.iris_b200_block_means(ptr(self.qm), None, ptr(self.q), heads * D, seq, heads, D, qb, None)
            rc |= lib.iris_b200_block_means(ptr(self.km), None, ptr(self.k), heads * D, seq, heads, D, kb, None)
            rc |= lib.iris_b200_block_select(ptr(self.lists), ptr(self.qm), ptr(self.km), None, nq, nk, heads, heads, D, topk, 1, 0)
            rc |= lib.iris_b200_attention_blocks(ptr(self.out), heads * D, ptr(self.q), heads * D, ptr(self.k),
                                                 heads * D, ptr(self.x, 2 * heads * D), ld, seq, seq, heads, heads, D, D ** -0.5, None,
                                                 ptr(self.lists), topk, qb, kb, AUTO)
            assert rc == 0

    a, b = Run(1), Run(2)
    side = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for r, s in zip((a, b), side):
        with torch.cuda.stream(s):
            r()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            r()
        graphs.append(g)
    for r, seed in ((a, 11), (b, 12)):
        r.x.copy_(randn(seed, seq, 3 * heads * D))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    got = [(r.lists.clone(), r.out.clone()) for r in (a, b)]
    for r, (lists, out) in zip((a, b), got):
        r()                                  # eager, on the module's stream again
        torch.cuda.synchronize()
        assert torch.equal(r.lists, lists) and torch.equal(r.out, out)
    done(lib)
