"""norm_rope_append where ends lie past the packed rows: they count as the rows'
own end, as in the attention, so that a request's last row is its newest token."""

from __future__ import annotations

import pytest
import torch

from _prefix import SCALE, api, call_norm, check_attention, check_norm, i32, norm_inputs

pytestmark = pytest.mark.gpu


def _run(d):
    got = {k: None if v is None else v.cuda() for k, v in d.items()}
    call_norm(got)
    torch.cuda.synchronize()
    got = {k: None if v is None else v.cpu() for k, v in got.items()}
    check_norm(got, d)
    return got


@pytest.mark.parametrize("ends", [[6, 99], [6, 2 ** 31 - 1], [6, 13], [40, 41], [-3, 12]])
@pytest.mark.parametrize("nope", [0, 8])
def test_ends_past_the_rows(ends, nope):
    print(f"ENDS {ends} {nope}", flush=True)
    d = norm_inputs([6, 6], [0, 130], 2, nope, torch.bfloat16, 11)
    d["ends"] = i32(ends)
    _run(d)


def test_the_attention_counts_the_same_rows():
    """Rows that were written are those that the rows see."""
    d = norm_inputs([6, 6], [20, 130], 4, 0, torch.bfloat16, 12)
    d["ends"][1] = 400
    got = _run(d)
    g = torch.Generator().manual_seed(13)
    c = {"query": torch.randn(12, 4, 512, generator=g).bfloat16(), "query_rope": got["query_rope"], "ends": d["ends"],
         "lengths": d["lengths"], "table": d["table"], "kv_cache": got["kv_cache"], "k_rope": got["k_rope"],
         "out": torch.zeros(12, 4, 512).bfloat16()}
    e = {k: v.cuda() for k, v in c.items()}
    api().shared_prefix_attention(e["query_rope"], e["query"], e["ends"], e["lengths"], e["table"], e["k_rope"], e["kv_cache"],
                                  SCALE, e["out"])
    check_attention(e["out"].cpu(), c)
