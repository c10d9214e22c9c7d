"""Forks and compactions whose copies fail: accounting, names and running requests stay as they were, and the engine goes on."""

import pytest

from test_host_long_lived import drain, engine

from minillm.engine.core import AddRequest

PROMPTS = {"a": list(range(3, 24)), "b": list(range(3, 20)) + [90], "c": [5, 6, 7] * 9}


class Failed(RuntimeError):
    pass


def started(**kw):
    core, outs = engine(**kw), {}
    for name, prompt in PROMPTS.items():
        core.add_request(AddRequest(name, prompt, 9))
    for _ in range(3):
        for o in core.step().outputs:
            outs.setdefault(o.req_id, []).extend(o.new_token_ids)
    return core, outs


def state(core):
    blocks, prefix = core.blocks, core.prefix
    return (blocks.num_free, blocks.num_cached, blocks._holders.tolist(), blocks._ticket.tolist(), dict(prefix._block_by_name),
            [n for n in prefix._name_by_block if n], [(r.req_id, list(r.block_ids)) for r in core.scheduler.running])


def failing(core, monkeypatch, error):
    def copy_blocks(src, dst):
        raise error

    monkeypatch.setattr(core.cache, "copy_blocks", copy_blocks)


@pytest.mark.parametrize("error", [Failed("a launch"), ValueError("a page"), KeyboardInterrupt()], ids=lambda e: type(e).__name__)
def test_a_fork_whose_copy_fails(monkeypatch, error):
    core, outs = started()
    free, cached, running = core.blocks.num_free, core.blocks.num_cached, list(core.scheduler.running)
    with monkeypatch.context() as m:
        failing(core, m, error)
        with pytest.raises(type(error)):
            core.fork("a", "d")
    core.check_blocks()
    assert (core.blocks.num_free, core.blocks.num_cached, core.scheduler.running) == (free, cached, running)
    core.fork("a", "d")  # the name is free
    drain(core, outs)
    plain, want = started()
    drain(plain, want)
    assert {k: v for k, v in outs.items() if k != "d"} == want and outs["d"] == want["a"][-len(outs["d"]):]


@pytest.mark.parametrize("error", [Failed("a launch"), ValueError("a page")], ids=lambda e: type(e).__name__)
def test_a_compaction_whose_copy_fails(monkeypatch, error):
    core, outs = started()
    core.abort("a")  # leaves gaps and idle names
    core.blocks.clear_cache()
    before = state(core)
    with monkeypatch.context() as m:
        failing(core, m, error)
        with pytest.raises(type(error)):
            core.compact()
    core.check_blocks()
    assert state(core) == before
    assert core.blocks.gaps() and state(core) == before  # looking moves nothing
    core.compact()
    assert core.blocks.gaps() == []
    drain(core, outs)
    plain, want = started()
    plain.abort("a")
    drain(plain, want)
    assert outs == want
