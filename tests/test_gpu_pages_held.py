"""A page of someone else that most places of a very large table name."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences,places", [(1024, 20000), (2048, 32768)])   # more than 2^24 places; as many as a table may have
def test_all_places_give_a_held_page_up(pkg, sequences, places):
    i32 = torch.int32
    table = torch.full((sequences, places), 1, dtype=i32, device="cuda")
    length = torch.full((sequences,), places * 16, dtype=i32, device="cuda")
    pool = torch.zeros((3, 1, 16, 8), dtype=torch.bfloat16, device="cuda")
    cache = pkg.PagedCache(pool, pool.clone(), table, length)
    refs = torch.tensor([0, -5, 0], dtype=i32, device="cuda")
    # all become children of the first, which names it as often as they did, and then end
    moves, counts = pkg.op_paged_fork(cache, refs, parent=torch.zeros(sequences, dtype=i32, device="cuda"))
    assert counts.tolist() == [0, 0] and refs.tolist() == [0, -5, 0] and bool((table == 1).all())
    moves, counts = pkg.op_paged_fork(cache, refs, parent=torch.full((sequences,), -1, dtype=i32, device="cuda"))
    assert counts.tolist() == [0, 0] and bool((moves == -1).all())
    assert refs.tolist() == [0, -5, 0]
    assert bool((table == -1).all()) and bool((length == 0).all())
    # and name it again, from a table of someone's own
    table[0].fill_(1)
    length[0] = places * 16
    pkg.op_paged_fork(cache, refs, parent=torch.zeros(sequences, dtype=i32, device="cuda"))
    assert refs.tolist() == [0, -5, 0] and bool((table == 1).all())
