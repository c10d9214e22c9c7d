"""Resident block tables follow lists of block ids that are cut and grow again (the uploads applied on the host)."""

import random

import pytest

from minillm.attention.metadata import DeviceBlockTables, SeqStep
from minillm.engine.block_manager import BlockManager


class Mirror:
    """A DeviceBlockTables and what its uploads leave on the device."""

    def __init__(self, rows, width):
        self.tables, self.width = DeviceBlockTables(rows, width, "cpu"), width
        self.held = [0] * (rows * width)
        self.uploads = 0

    def step(self, lists):
        rows, updates = self.tables.sync(list(lists), [SeqStep(0, 1, ids) for ids in lists.values()])
        for at, block in zip(updates[::2], updates[1::2]):
            self.held[at] = block
        self.uploads = len(updates) // 2
        for row, ids in zip(rows, lists.values()):
            assert self.held[row * self.width:row * self.width + len(ids)] == ids


@pytest.mark.parametrize("grow", [0, 1, 2, 3])
def test_a_list_cut_and_grown_again_is_uploaded(grow):
    # five blocks, cut to three and grown by fewer, as many and more: other blocks than before lie behind the third
    blocks, mirror = BlockManager(12, 16), Mirror(2, 8)
    table = blocks.allocate(5)
    mirror.step({"a": table})
    blocks.trim(table, 40)
    table += blocks.allocate(grow)
    mirror.step({"a": table})
    assert mirror.uploads == grow
    mirror.step({"a": table})
    assert mirror.uploads == 0


def test_the_last_block_alone_does_not_tell():
    # cut to one block and grown to the old length, with the old last block in its old place
    blocks, mirror = BlockManager(4, 16), Mirror(1, 4)
    table = blocks.allocate(3)  # 0 1 2
    mirror.step({"a": table})
    blocks.trim(table, 16)
    other = blocks.allocate(1) + blocks.allocate(1)  # 3, 2
    blocks.free(other[:1])
    table += [3, 2]
    assert len(table) == 3
    mirror.step({"a": table})


def test_every_mirror_follows_and_rows_that_sit_out_do_too():
    blocks, mirrors = BlockManager(20, 16), [Mirror(3, 6), Mirror(3, 6)]
    lists = {k: blocks.allocate(4) for k in "ab"}
    for m in mirrors:
        m.step(lists)
    blocks.trim(lists["b"], 16)
    for m in mirrors:
        m.step({"a": lists["a"]})
        assert m.uploads == 0
    lists["b"] += blocks.allocate(3)
    for m in mirrors:
        m.step(lists)
        assert m.uploads == 3


@pytest.mark.parametrize("seed", range(5))
def test_lists_that_change_at_random(seed):
    rng = random.Random(seed)
    blocks, mirror, lists = BlockManager(40, 16), Mirror(6, 10), {}
    for i in range(300):
        what = rng.random()
        if what < 0.3 and len(lists) < 6 and blocks.num_free > 10:
            lists[i] = blocks.allocate(rng.randint(1, 6))
        elif lists:
            key = rng.choice(list(lists))
            ids = lists[key]
            if what < 0.5:
                blocks.trim(ids, rng.randint(1, 16 * len(ids)))
            elif what < 0.8 and len(ids) < 10 and blocks.num_free > 4:
                ids += blocks.allocate(rng.randint(1, min(4, 10 - len(ids))))
            elif what < 0.87:
                lists[key] = list(ids)  # a new list of the same blocks, as after a compaction
            elif what < 0.93:
                blocks.free(lists.pop(key))
                mirror.tables.release(key)
        if lists and rng.random() < 0.6:
            mirror.step({k: lists[k] for k in rng.sample(list(lists), rng.randint(1, len(lists)))})
        blocks.check(list(lists.values()))


def test_a_cut_through_a_shared_block_is_refused():
    # its next tokens would go into the other table's block; at a block's end, or behind a copy, nothing is shared
    blocks = BlockManager(10, 16)
    table = blocks.allocate(4)
    child, copies = blocks.fork(table, 64)
    assert child == table and copies == []
    for t in (table, child):
        with pytest.raises(ValueError, match="shared"):
            blocks.trim(t, 40)
        assert len(t) == 4
    blocks.check([table, child])
    blocks.trim(child, 32)
    own, copies = blocks.fork(table, 40)
    blocks.trim(own, 33)
    blocks.check([table, child, own])
    blocks.free(child), blocks.free(own)
    blocks.trim(table, 40)
    blocks.check([table])
    with pytest.raises(ValueError, match="shared"):
        other, _ = blocks.fork(table, 48)
        blocks.trim(other, 47)  # within its last block, with none to release


def test_a_block_that_is_cut_loses_its_name():
    from minillm.cache.prefix import PrefixCache

    prefix = PrefixCache()
    blocks = BlockManager(6, 16, prefix)
    table = blocks.allocate(3)
    for i, b in enumerate(table):
        prefix.insert(b"%d" % i, b)
    blocks.trim(table, 20)
    assert prefix.lookup([b"0", b"1"]) == table[:1] and blocks.num_cached == 1  # the third, whole and idle
    blocks.check([table])
    blocks.trim(table, 16)
    assert prefix.lookup([b"0"]) == table
    blocks.check([table])


def test_fewer_than_no_tokens():
    blocks = BlockManager(6, 16)
    table = blocks.allocate(3)
    for n in (-1, -16, -40):
        for call in (lambda: blocks.fork(table, n), lambda: blocks.trim(table, n)):
            with pytest.raises(ValueError, match="tokens"):
                call()
    assert len(table) == 3 and blocks.num_free == 3
    blocks.check([table])
