"""The producer warp of the tensor-core attention over key blocks, its own source run on host threads
(host/attn_blocks_producer.cpp): every copy that it issues is waited for by somebody before the CTA can leave, and the key
tiles that it puts together hold the keys of the lists. No device."""
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SOURCE = os.path.join(os.path.dirname(HERE), "iris.c_b200", "csrc", "attn_blocks_sm100.cu")


@pytest.fixture(scope="module")
def producer(tmp_path_factory):
    text = open(SOURCE).read()
    first, behind = text.index("static constexpr int kThreads"), text.index("/* Rows of V whose key does not count")
    folder = tmp_path_factory.mktemp("producer")
    part, exe = folder / "producer.inc", folder / "producer"
    part.write_text(text[first:behind])
    subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", "-w", '-DPRODUCER_INC="%s"' % part, "-o", str(exe),
                    os.path.join(HERE, "host", "attn_blocks_producer.cpp")], check=True)

    def run(seq_q, seq_k, heads, q_block, k_block, lists, mask=None, group=1, rank=0, parts=1, part_len=None, block=0, grid=1, give_up=0):
        """lists [heads][q_blocks][n]; the loads of Q, K and V, and the products
        with K and V, as {name: (issued, waited)}, and the query tiles of the CTA: for
        each its key tiles as 128 key rows, None where the key does not count."""
        n = len(lists[0][0])
        args = [seq_q, seq_k, heads, group, n, q_block, k_block, rank, parts, n if part_len is None else part_len, block, grid, give_up]
        args += [b for head in lists for row in head for b in row] + (list(mask) if mask is not None else [])
        done = subprocess.run([str(exe)] + [str(x) for x in args], capture_output=True, text=True, timeout=300)
        assert done.returncode == 0, (done.returncode, done.stderr)
        unit = min(k_block, 128)
        loads, records, boxes = {}, [], {"Q": [], "K": [], "V": []}
        for line in done.stdout.splitlines():
            w = line.split()
            if w[0] in ("copies", "products"):
                loads[w[1] if w[0] == "copies" else w[1] + " products"] = (int(w[3]), int(w[5]))
            elif w[0] == "box":
                boxes[w[1]].append(tuple(int(x) for x in w[2:]))
            else:
                records.append(w)
        places = {"Q": 0, "K": 32768, "V": 65536}
        keys = []                            # of every key tile: the row at each place
        for t in "KV":
            tiles = {}
            for load, x, row, at in boxes[t]:
                half, first = divmod((at - places[t]) // 128, 128)
                assert x % 64 == 0 and x // 64 % 2 == half and at % (unit * 128) == 0
                rows = tiles.setdefault(load, [{}, {}])[half]
                for i in range(unit):
                    assert rows.setdefault(first + i, (x // 128, row + i)) == (x // 128, row + i)
            assert all(a == b for a, b in tiles.values())              # both halves of a head hold the same rows
            keys.append([tiles[i][0] for i in range(len(tiles))])
        assert keys[0] == keys[1] or (give_up and keys[0][:len(keys[1])] == keys[1])
        out, j = [[]], 0
        for r in records:
            if r[0] == "end":
                out.append([])
                continue
            bits = [int(b, 16) for b in r[2:]]
            valid = [bits[i // 32] >> (i % 32) & 1 for i in range(128)]
            assert (r[1] == "whole") == all(valid)
            if j < len(keys[0]):             # (a record whose copies were not issued any more)
                out[-1].append([keys[0][j][i] if v else None for i, v in enumerate(valid)])
            j += 1
        assert give_up or (out.pop() == [] and j == len(keys[0]))
        return loads, out

    return run


def all_waited(loads):
    return all(issued == waited for issued, waited in loads.values())


EMPTY = [-1, 99, -5]
KEYS = [0, 2, -1]


@pytest.mark.parametrize("rows", [[EMPTY], [KEYS, EMPTY], [EMPTY, KEYS, EMPTY, EMPTY], [EMPTY, KEYS], [KEYS]])
def test_no_copy_outlives_the_cta(producer, rows):
    """The last query tile of a CTA may have no usable key: its Q is on its way by then and has to arrive before the CTA leaves."""
    loads, tiles = producer(128 * len(rows), 300, 1, 128, 64, [rows])
    assert len(tiles) == len(rows) and [bool(t) for t in tiles] == [r is KEYS for r in rows]
    assert loads["Q"][0] == len(rows)
    assert all_waited(loads), loads


def test_no_copy_outlives_the_cta_with_masked_keys(producer):
    """Lists whose blocks are masked as a whole, in one CTA and in every part of a cluster."""
    mask = [1] * 64 + [0] * 128 + [1] * 64
    for rank, keys in ((0, True), (1, False), (2, False)):
        loads, tiles = producer(100, 256, 1, 128, 64, [[[0, 0, 1, 2, 2, 1]]], mask, rank=rank, parts=3, part_len=2, block=rank,
                                    grid=3)
        assert [bool(t) for t in tiles] == [keys] and all_waited(loads), (rank, loads)


@pytest.mark.parametrize("k_block,n,masked,step", [(16, 9, False, 1), (16, 40, True, 1), (32, 7, True, 2), (64, 5, False, 1), (64, 35, True, 3),
                                                   (128, 3, True, 1), (384, 2, True, 2), (256, 2, False, 1)])
def test_key_tiles_hold_the_keys_of_the_lists(producer, k_block, n, masked, step):
    """Every key of the lists once, in their order, whatever is masked, missing or not there; several heads and query tiles."""
    rng = random.Random(k_block + n)
    seq_q, seq_k, heads, group, q_block = 300, 700, 2, 2, 200
    nk = -(-seq_k // k_block)
    mask = [int(rng.random() < 0.8) and not 256 <= r < 384 for r in range(seq_k)] if masked else [1] * seq_k
    mask = [int(m) for m in mask]
    lists = [[[rng.choice([rng.randrange(nk), rng.randrange(nk), -1, nk, 2 ** 31 - 1]) for _ in range(n)] for _ in range(2)]
             for _ in range(heads)]
    lists[1][0] = [-1] * n
    per_head = 4                             # two query blocks of two tiles; the second block has one that does not exist
    for block in range(step):
        loads, tiles = producer(seq_q, seq_k, heads, q_block, k_block, lists, mask if masked else None, group=group, block=block,
                                grid=step)
        assert all_waited(loads), loads
        items = list(range(block, heads * per_head, step))
        assert len(tiles) == len(items)
        for item, got in zip(items, tiles):
            head, in_head = divmod(item, per_head)
            qb, tile = divmod(in_head, 2)
            exists = qb * q_block + tile * 128 < seq_q
            want = [(head // group, r) for b in lists[head][qb] if 0 <= b < nk
                    for r in range(b * k_block, min(seq_k, (b + 1) * k_block)) if mask[r]] if exists else []
            assert [k for t in got for k in t if k is not None] == want


@pytest.mark.parametrize("give_up", range(1, 9))
def test_no_copy_outlives_a_cta_that_gives_up(producer, give_up):
    """The other warps stop at any record, the last ones among them: the copies that nobody waits for any more are drained."""
    loads, _ = producer(128 * 3, 1000, 1, 128, 64, [[[0, 1, 2, 3, 4], [5, 6, -1, -1, -1], [7, 8, 9, 10, 11]]], give_up=give_up)
    assert loads["K"][0] >= 1 and all(loads[t][0] == loads[t][1] for t in "QKV"), loads
