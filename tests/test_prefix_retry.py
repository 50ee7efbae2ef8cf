"""A pages_branch call that lacks pages, and how it is repeated: the rows have
taken over their parents' tables, so the parents are not named again."""

from __future__ import annotations

from pathlib import Path

import pytest
import torch

from _prefix import api, i32, make_pages
from oracle import prefix_oracle as O

LENGTHS, NEW, SWAP = [130, 260, 300], [200, 300, 0], [1, 0, 2]


def _start(batch=3, cols=6, spare=2):
    """Rows 0 and 1 go on from each other; row 2 holds what they will need."""
    lengths = LENGTHS + [0] * (batch - 3)
    table, refs = make_pages(lengths, 8 + spare, cols, 9)
    return lengths, table, refs


def _serve(branch, lengths, table, refs):
    """What the interface says a caller does: the states after each of the three calls."""
    batch = len(lengths)
    new, parents = NEW + [0] * (batch - 3), SWAP + list(range(3, batch))
    states = [branch(lengths, new, table, refs, parents)]
    ends = [b if b != 2 else -1 for b in range(batch)]
    states.append(branch(*states[-1][:1], [0] * batch, *states[-1][1:3], ends))
    states.append(branch(*states[-1][:1], new, *states[-1][1:3], None))
    return states


def _check(states, lengths, table, refs):
    batch = len(lengths)
    failed, freed, served = states
    none = [(-1, -1, 0)] * batch
    # Taken over, but nobody has new pages, and nothing is to be copied.
    assert failed[4] > 0 and failed[3] == none
    assert failed[0][:3] == [260, 130, 300]
    assert failed[1] == [table[1], table[0]] + table[2:] and failed[2] == refs
    assert freed[0][:3] == [260, 130, 0] and freed[1][2] == [-1] * len(table[2]) and freed[4] == 0
    # As one call with the parents would have it, had the pages been free before.
    first = O.branch(lengths, [0] * batch, table, refs, [b if b != 2 else -1 for b in range(batch)])
    want = O.branch(first[0], NEW + [0] * (batch - 3), first[1], first[2], SWAP + list(range(3, batch)))
    assert served == want and want[4] == 0
    assert served[1][0][:3] == table[1][:3] and served[1][1][:2] == table[0][:2]


def _on_gpu(lengths, new, table, refs, parents):
    d = [i32(v).cuda() for v in (lengths, new, table, refs)]
    out = [torch.full((len(lengths),), 99, dtype=torch.int32, device="cuda") for _ in range(3)]
    missing = torch.full((1,), 99, dtype=torch.int32, device="cuda")
    api().pages_branch(*d, *out, missing, parents=None if parents is None else i32(parents).cuda())
    torch.cuda.synchronize()
    return d[0].tolist(), d[2].tolist(), d[3].tolist(), list(zip(*[o.tolist() for o in out])), missing.item()


def test_a_call_that_lacks_pages_is_repeated_without_parents():
    start = _start()
    _check(_serve(O.branch, *start), *start)


def test_the_same_parents_again_would_be_applied_twice():
    lengths, table, refs = _start()
    failed = O.branch(lengths, NEW, table, refs, SWAP)
    again = O.branch(failed[0], NEW, failed[1], failed[2], SWAP)
    assert again[4] > 0 and again[0] == lengths and again[1] == table


def test_the_interface_says_so():
    header = (Path(__file__).resolve().parents[1] / "include" / "nvdsa_ext.h").read_text()
    branch = header[:header.index("nvdsa_pages_branch_workspace_size")].rpartition("/*")[2]
    for text, how in ((api().pages_branch.__doc__, "parents=None"), (branch, "parents NULL")):
        assert how in text and "repeated" in text and "free for the next." not in " ".join(text.split())


@pytest.mark.gpu
@pytest.mark.parametrize("batch,cols", [(3, 6), (100, 6)])
def test_a_call_that_lacks_pages_on_the_gpu(batch, cols):
    """By one workgroup, and with tables that are taken over before."""
    start = _start(batch, cols)
    print(f"RETRY {batch}", flush=True)
    _check(_serve(_on_gpu, *start), *start)
