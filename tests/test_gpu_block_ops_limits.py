"""The attention over key blocks when one of its bounded waits runs out, on the GPU: the call reports it, whatever was under way
has ended, and the calls that follow are right."""
import pytest
import torch

import block_ops_ref as ref
from test_gpu_block_ops import AUTO, D, TCGEN05, done, lib, ptr, randn      # noqa: F401 (lib is a fixture)

pytestmark = pytest.mark.gpu

ETIMEOUT = 3


class Call:
    """Lists of `skip` entries that name nothing and then two blocks: reading them takes the producer skip / 32 loads one after
    the other, while the other warps wait for a first key tile."""

    def __init__(self, sq, heads, skip, seed=0):
        self.sq, self.heads, self.sk, self.qb, self.kb = sq, heads, 512, 128, 64
        nq = -(-sq // self.qb)
        self.q, self.k, self.v = (randn(seed + i, r, c).bfloat16() for i, (r, c) in
                                  enumerate([(sq, heads * D), (self.sk, D), (self.sk, D)]))
        self.short = torch.tensor([1, 6], dtype=torch.int32).expand(heads, nq, 2)
        lists = torch.full((heads, nq, skip + 2), -1, dtype=torch.int32)
        lists[..., skip:] = self.short
        self.gpu = [t.cuda() for t in (self.q, self.k, self.v, lists)]
        self.out = torch.zeros(sq + 1, heads * D, dtype=torch.bfloat16, device="cuda")

    def launch(self, lib, mask=None):
        q, k, v, lists = self.gpu
        self.out.fill_(7.0)
        assert lib.iris_b200_attention_blocks(ptr(self.out), self.heads * D, ptr(q), self.heads * D, ptr(k), D, ptr(v), D, self.sq,
                                              self.sk, self.heads, 1, D, D ** -0.5, ptr(mask), ptr(lists), lists.shape[2], self.qb,
                                              self.kb, TCGEN05) == 0

    def check(self):
        if not hasattr(self, "want"):
            self.want = ref.attention(self.q, self.k, self.v, self.heads, 1, D, D ** -0.5, None, self.short, self.qb, self.kb)
        want, mag = self.want
        got = self.out[:self.sq].cpu().double()
        assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mag).all()
        assert (self.out[self.sq] == 7).all()


def status(lib):
    rc = lib.iris_b200_check_device_status()
    lib.iris_b200_clear_error()
    return rc


@pytest.mark.parametrize("sq,heads,skip", [(128, 1, 1 << 20), (300, 3, 1 << 20), (1000, 40, 1 << 17)])
def test_wait_that_runs_out_is_reported_and_the_next_call_is_fine(lib, sq, heads, skip):
    """One tile in a cluster, several clusters, more tiles than CTAs. The limit is 5 us, looked at every 0.7 ms (64 tries); the
    wait for the first keys takes 1.7 ms."""
    call = Call(sq, heads, skip)
    try:
        for _ in range(3):
            lib.iris_b200_set_wait_limit_us(5)
            call.launch(lib)
            assert status(lib) == ETIMEOUT
            assert (call.out[sq] == 7).all()
            lib.iris_b200_set_wait_limit_us(0)
            call.launch(lib)
            assert status(lib) == 0
            call.check()
    finally:
        lib.iris_b200_set_wait_limit_us(0)
    done(lib)


def test_limits_of_the_length_of_a_copy(lib):
    """Limits near the time that a copy or a product takes: a call is right or says that a wait ran out, and the next is right."""
    call = Call(1000, 40, 30)
    other = Call(260, 2, 0, seed=9)
    try:
        for us in (1, 2, 3, 5, 8, 12, 20) * 3:
            lib.iris_b200_set_wait_limit_us(us)
            call.launch(lib)
            rc = status(lib)
            assert rc in (0, ETIMEOUT)
            if rc == 0:
                call.check()
            lib.iris_b200_set_wait_limit_us(0)
            other.launch(lib)
            assert status(lib) == 0
            other.check()
    finally:
        lib.iris_b200_set_wait_limit_us(0)
    call.launch(lib)
    done(lib)
    call.check()


@pytest.mark.parametrize("skip,masked", [(1 << 25, False), (1 << 21, True)])
def test_reading_a_list_may_take_longer_than_the_limit(lib, skip, masked):
    """Tens of milliseconds of entries that name nothing, or a block that is masked as a whole, under a limit of ten: the
    other warps see that the producer reads on."""
    call = Call(100, 1, skip)
    mask = None
    if masked:
        call.gpu[3][..., :skip] = 3
        mask = torch.ones(call.sk, dtype=torch.int32)
        mask[3 * call.kb:4 * call.kb] = 0
        mask = mask.cuda()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    try:
        lib.iris_b200_set_wait_limit_us(10000)
        for _ in range(2):
            a.record()
            call.launch(lib, mask)
            b.record()
            assert status(lib) == 0
            assert a.elapsed_time(b) > 20.0
            call.check()
    finally:
        lib.iris_b200_set_wait_limit_us(0)
    done(lib)
