"""A cache in eight bits, as far as it goes without a GPU: a context that comes back with other lengths, refusals, room for cut tiles."""
import pytest
import torch

from synaptix_b200 import ops
from synaptix_b200.cache import Cache, KVRequest
from synaptix_b200.cache.store import BundleRequest, StateRequest
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


@pytest.mark.parametrize("others_first", [False, True])
@pytest.mark.parametrize("bundled", [False, True])
def test_a_request_that_cannot_be_held_in_eight_bits_is_refused_beside_an_equal_one_that_can(others_first, bundled):
    takes, does_not = KVRequest(2, 64, eight_bit=True), KVRequest(2, 64)
    state = StateRequest((4,), torch.float32)
    requests = [takes, BundleRequest((state, BundleRequest((does_not,)))) if bundled else does_not]
    if others_first:
        requests.reverse()
    kw = dict(max_tokens=64, max_seqs=1, dtype=torch.bfloat16, device="cpu")
    with pytest.raises(ValueError, match="eight bits"):
        Cache(requests, kv_dtype="fp8", **kw)
    assert len(Cache(requests, **kw).kv_groups) == 1                  # (in the compute dtype they share a group)
    assert len(Cache([takes, BundleRequest((state, takes))], kv_dtype="fp8", **kw).kv_groups) == 1


def test_places_of_cut_tiles():
    from synaptix_b200.ops.attention import tc_part_rows
    tiles = [(0, 99), (100000, 100063), (0, 127), (128, 128), (5000, 5009), (700, 827)]
    assert tc_part_rows(tiles, 261, None) == ([-1, 0, -1, -1, -1, -1], 3 * 64)                # 782 blocks in three
    assert tc_part_rows(tiles, 2, None) == ([-1, 0, -1, -1, 391 * 64, 391 * 64 + 20 * 10],
                                            391 * 64 + 20 * 10 + 4 * 128)
    # a window of 200: keys 99,801 to 100,063 are blocks 779 to 781; 4,801 to 5,009 37 to 39; 501 to 827 3 to 6
    assert tc_part_rows(tiles, 2, 200) == ([-1, 0, -1, -1, 2 * 64, 2 * 64 + 2 * 10], 2 * 64 + 2 * 10 + 2 * 128)
    assert tc_part_rows([], 1, None) == ([], 0)
