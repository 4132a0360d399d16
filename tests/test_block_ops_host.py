"""Host side of the multi-axis rotation, the block lists and the attention over
them: the rotation plan against its definition, and every refusal. No device."""
import ctypes as C
import math
from fractions import Fraction

import pytest

import __graft_entry__ as ge

EINVAL, ENODEV, EUNSUPPORTED = 1, 4, 6
P = 4096                                    # a pointer that no refused call follows


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(os.path.join(ge.PKG_DIR, "libiris_b200.so")):
        ge.build()
    lib = ge.load_package().load()
    yield lib
    lib.iris_b200_clear_error()


def plan_rc(lib, dims, scales=None, theta=10000.0, one=False, hd=128, n=None):
    from iris_c_b200.binding import RopeAxes
    p = RopeAxes()
    d = (C.c_int * max(1, len(dims)))(*dims)
    s = (C.c_double * len(scales))(*scales) if scales else None
    return lib.iris_b200_rope_axes_plan(p, d, s, len(dims) if n is None else n, theta, int(one), hd), p


@pytest.mark.parametrize("dims,scales,theta,one,hd", [
    ((32, 32, 32, 32), None, 2000.0, False, 128), ((32, 48, 48), (2.5, 1.0, 1.0), 256.0, False, 128),
    ((16, 56, 56), (1.0, -0.5, 3.0), 1e6, True, 128), ((0, 10, 4), None, 10000.0, False, 64), ((512,), (24.0,), 500.0, False, 512),
])
def test_plan_holds_the_fractions_of_a_turn(lib, dims, scales, theta, one, hd):
    rc, p = plan_rc(lib, dims, scales, theta, one, hd)
    assert rc == 0 and p.n == len(dims) and p.head_dim == hd
    j = 0
    for a, dim in enumerate(dims):
        for i in range(dim // 2):
            power = 2.0 * j / hd if one else 2.0 * i / dim
            want = (scales[a] if scales else 1.0) * theta ** -power / (2 * math.pi)
            got = Fraction(p.turn[j], 1 << 64)
            off = abs(float(got - Fraction(want % 1.0)))
            # the double power is off by a few 2^-53 of its value
            assert min(off, 1.0 - off) <= 8 * 2.0 ** -53 * max(1.0, abs(want)) and p.axis[j] == a
            j += 1
    assert all(p.turn[i] == 0 for i in range(j, 256))


def test_plan_phase_of_far_positions(lib):
    """p * turn modulo 2^64 is the phase of the exact angle, for positions of either sign."""
    rc, p = plan_rc(lib, (128,), None, 10000.0)
    assert rc == 0
    for pos in (1, -1, 12345, -77777, 2 ** 31 - 1, -2 ** 31):
        for j in (0, 1, 17, 63):
            phase = (pos * p.turn[j]) % (1 << 64) / 2.0 ** 64
            want = pos * (10000.0 ** (-2.0 * j / 128)) / (2 * math.pi) % 1.0
            off = abs(phase - want)
            assert min(off, 1 - off) <= 2.0 ** -50 * abs(pos) + 2.0 ** -50


@pytest.mark.parametrize("kw", [
    dict(dims=(33,)), dict(dims=(-2, 4)), dict(dims=(64, 66)), dict(dims=(128,), theta=0.0), dict(dims=(128,), theta=-5.0),
    dict(dims=(128,), theta=math.inf), dict(dims=(128,), theta=math.nan), dict(dims=(64,), scales=(math.inf,)),
    dict(dims=(64,), hd=63), dict(dims=(64,), hd=514), dict(dims=(64,), hd=0), dict(dims=(2,) * 9), dict(dims=(), n=0),
])
def test_plan_refusals(lib, kw):
    assert plan_rc(lib, **kw)[0] == EINVAL
    lib.iris_b200_clear_error()


def refused(lib, code, rc):
    assert rc == code, rc
    assert lib.iris_b200_last_error() == code
    lib.iris_b200_clear_error()


def test_rotation_refusals(lib):
    _, plan = plan_rc(lib, (128,))

    def tables(cos=P, sin=P, pos=P, axes=plan, seq=4, hd=128):
        return lib.iris_b200_rope_axes_tables(cos, sin, pos, axes, seq, hd)

    def rows(qo=P, ldqo=512, ko=P, ldko=512, q=8192, k=9216, ldi=512, wq=None, wk=None, pos=P, axes=plan, seq=4, heads=2, kv=2,
             hd=128, eps=1e-6, split=0):
        return lib.iris_b200_qk_norm_rope_axes(qo, ldqo, ko, ldko, q, k, ldi, wq, wk, pos, axes, seq, heads, kv, hd, eps, split)

    for kw in (dict(cos=None), dict(sin=None), dict(pos=None), dict(axes=None), dict(seq=-1), dict(hd=64), dict(hd=127)):
        refused(lib, EINVAL, tables(**kw))
    broken = type(plan)()                   # never planned
    refused(lib, EINVAL, tables(axes=broken))
    odd = plan_rc(lib, (64, 64))[1]
    odd.axis[3] = 7                         # an axis that the rows have no position for
    refused(lib, EINVAL, tables(axes=odd))
    for kw in (dict(qo=None), dict(q=None), dict(k=None), dict(ko=None), dict(pos=None), dict(axes=None), dict(seq=-1),
               dict(heads=0), dict(kv=-1), dict(hd=64), dict(ldi=255), dict(ldqo=255), dict(ldko=255), dict(wq=P), dict(wk=P),
               dict(eps=-1.0), dict(eps=math.nan), dict(qo=8192, ldqo=520), dict(ko=9216, ldko=520)):
        refused(lib, EINVAL, rows(**kw))


def test_block_means_and_select_refusals(lib):
    def means(m=P, c=P, x=P, ldx=256, seq=9, heads=2, hd=128, block=4, mask=None):
        return lib.iris_b200_block_means(m, c, x, ldx, seq, heads, hd, block, mask)

    for kw in (dict(m=None), dict(x=None), dict(ldx=255), dict(seq=-1), dict(heads=0), dict(hd=0), dict(block=0), dict(block=-3)):
        refused(lib, EINVAL, means(**kw))

    def select(lst=P, qm=P, km=P, c=None, nq=3, nk=5, heads=4, kv=2, hd=128, topk=2, first=0, last=0):
        return lib.iris_b200_block_select(lst, qm, km, c, nq, nk, heads, kv, hd, topk, first, last)

    for kw in (dict(lst=None), dict(qm=None), dict(km=None), dict(nq=-1), dict(nk=-1), dict(heads=0), dict(kv=0), dict(kv=3),
               dict(hd=0), dict(topk=0), dict(first=-1), dict(last=-1), dict(first=2, last=1)):
        refused(lib, EINVAL, select(**kw))
    refused(lib, EUNSUPPORTED, select(nk=23553))
    refused(lib, EUNSUPPORTED, select(hd=513))


def test_attention_blocks_refusals(lib):
    def attn(out=P, ldo=512, q=P, ldq=512, k=P, ldk=512, v=P, ldv=512, sq=8, sk=8, heads=4, kv=2, hd=128, scale=0.1, mask=None, lst=P,
             n=2, qb=4, kb=4, kernel=0):
        return lib.iris_b200_attention_blocks(out, ldo, q, ldq, k, ldk, v, ldv, sq, sk, heads, kv, hd, scale, mask, lst, n, qb, kb,
                                              kernel)

    for kw in (dict(out=None), dict(q=None), dict(k=None), dict(v=None), dict(lst=None), dict(ldo=511), dict(ldq=511),
               dict(ldk=255), dict(ldv=255), dict(sq=-1), dict(sk=-1), dict(heads=0), dict(kv=0), dict(kv=3), dict(hd=0), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(n=-1), dict(qb=0), dict(kb=0), dict(kernel=3),
               dict(kernel=-1), dict(n=2 ** 30 + 1), dict(heads=65536, kv=1, hd=1, ldo=65536, ldq=65536)):
        refused(lib, EINVAL, attn(**kw))
    refused(lib, EUNSUPPORTED, attn(hd=64, kernel=1))          # outside the tensor-core kernel's domain
    refused(lib, EUNSUPPORTED, attn(kb=48, kernel=1))
    refused(lib, EUNSUPPORTED, attn(ldv=260, kb=64, kernel=1))


def test_good_arguments_need_a_device(lib):
    if lib.iris_dev_available():
        pytest.skip("a device is initialised")
    _, plan = plan_rc(lib, (128,))
    refused(lib, ENODEV, lib.iris_b200_rope_axes_tables(P, P, P, plan, 4, 128))
    refused(lib, ENODEV, lib.iris_b200_qk_norm_rope_axes(P, 256, P, 256, 2 * P, 3 * P, 256, None, None, P, plan, 4, 2, 2, 128,
                                                         1e-6, 0))
    refused(lib, ENODEV, lib.iris_b200_block_means(P, P, P, 256, 9, 2, 128, 4, None))
    refused(lib, ENODEV, lib.iris_b200_block_select(P, P, P, None, 3, 5, 4, 2, 128, 2, 0, 0))
    refused(lib, ENODEV, lib.iris_b200_attention_blocks(P, 512, P, 512, P, 512, P, 512, 8, 8, 4, 2, 128, 0.1, None, P, 2,
                                                         4, 4, 0))
