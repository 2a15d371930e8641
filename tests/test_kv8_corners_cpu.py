"""A cache in eight bits, as far as it goes without a GPU: a context that comes back with other lengths."""
import torch

from synaptix_b200 import ops
from test_kv8_cpu import step


def comes_back(ctx, lens, new):
    """The same context (and what was made for it) with other lengths, in new lists or in the same ones."""
    for name, value in vars(step(lens, new)).items():
        if name not in ("scratch", "host"):
            setattr(ctx, name, value)
    for name, value in step(lens, new).host.items():
        ctx.host[name][:] = value
    return ctx


def test_what_is_made_of_a_steps_lengths_is_made_anew_for_others():
    ctx, fresh = step([300, 200], [300, 200]), step([600, 700], [200, 300])
    for rows in (64, 128):
        assert ops._query_tiles(ctx, rows, torch.device("cpu"))[0].tolist() == [0] * -(-300 // rows) + [1] * -(-200 // rows)
    assert [list(x) for x in ops._portions(ctx)] == [[0, 300, 500], [0, 0]]
    kept = ops._portions(ctx), ops._query_tiles(ctx, 64, torch.device("cpu"))
    assert all(a is b for a, b in zip(kept, (ops._portions(ctx), ops._query_tiles(ctx, 64, torch.device("cpu")))))
    comes_back(ctx, [600, 700], [200, 300])
    assert ctx.scratch
    for rows in (64, 128):
        for got, want in zip(ops._query_tiles(ctx, rows, torch.device("cpu")), ops._query_tiles(fresh, rows, torch.device("cpu"))):
            assert torch.equal(got, want)
    assert [list(x) for x in ops._portions(ctx)] == [[0, 200, 500], [400, 400]]
    ctx.host["seq_past"] = [1, 2]
    assert list(ops._portions(ctx)[1]) == [1, 2]
