"""A check of the attention over many keys that notices a page.

Element by element, an output may be off by half a step of sum p |v - o|, which over
N keys of one size is sqrt(N) times the output itself: a bound of that kind passes
outputs that lack half of the keys.  But roundings are as good as independent, and a
row's 512 dims meet the same ones, so that over the dims of a (row, head) the root
mean square of what they do is that of independent errors."""

from __future__ import annotations

import torch

from _prefix import HALF_STEP, PAGE, SCALE, i32, make_cache, make_queries
from oracle import prefix_oracle as O


class Check:
    """The 64-bit output of a call on its tensors' device, and the root mean square over
    the dims of what may separate another from it, for every (row, head).

    Each term takes its largest rounding, where the root mean square of a uniform one is
    0.58 of it: the store's half step; half a step of each weight, times its value's
    distance from the output, added as squares; a sum of n fp32 terms sqrt(n) 2^-24 of
    their magnitudes: the output's and the weights' n keys, and the scores' 576 products,
    which move a weight by their error."""

    def __init__(self, c, scale=SCALE):
        self.c, self.rows = c, int(c["ends"][-1])
        step, pages = HALF_STEP[c["kv_cache"].dtype], c["kv_cache"].shape[0]
        rms = lambda x: x.square().mean(-1).sqrt()  # noqa: E731
        q = torch.cat([c["query"], c["query_rope"]], -1).double()
        self.want = torch.zeros_like(c["query"], dtype=torch.float64)
        self.tolerance = torch.zeros_like(self.want[..., 0])
        start = 0
        for b, end in enumerate(c["ends"].tolist()):
            n = int(c["lengths"][b])
            at = c["table"][b, : -(-n // PAGE)].long()
            assert bool(((at >= 0) & (at < pages)).all())
            keys = torch.cat([c["kv_cache"][at].flatten(0, 2), c["k_rope"][at].flatten(0, 2)], -1)[:n].double()
            for t in range(start, end):
                seen = keys[: n - (end - 1 - t)]
                values, turned = seen[:, :512].contiguous(), seen.T.contiguous()
                p = torch.softmax(q[t] @ turned * scale, -1)
                o, squares = p @ values, p.square()
                apart = squares @ values.square() - 2 * o * (squares @ values) + squares.sum(-1, keepdim=True) * o.square()
                reach = (q[t].abs() @ turned.abs()).amax(-1) * abs(scale)
                sums = 2.0 ** -24 * (2 * len(seen) ** 0.5 + 24 * reach + 4)
                self.want[t] = o
                self.tolerance[t] = step * rms(o) + step * apart.mean(-1).clamp(min=0).sqrt() + sums * rms(p @ values.abs())
            start = end

    def worst(self, got):
        """The largest distance over its tolerance, of any row and head."""
        off = (got.double() - self.want)[:self.rows].square().mean(-1).sqrt()
        return float((off / self.tolerance[:self.rows]).max())


def many_keys(heads, dtype, tokens=131072, rows=1):
    """One request over as many slots as parts and windows of pages take."""
    return make_queries(make_cache([], [], [tokens], 70, dtype, size=0.5), [rows], heads, 71, size=0.5)


def two_on_a_prefix(heads, dtype, pages=1100):
    """A prefix of more pages than are held at a time."""
    return make_queries(make_cache([pages * PAGE], [2], [3, 150], 72, dtype), [1, 1], heads, 73)


def batch_on_a_prefix(heads, dtype, requests=33, pages=130):
    """Read once: the prefix's items and the requests' own."""
    own = [(i * 37) % 300 for i in range(requests)]
    return make_queries(make_cache([pages * PAGE], [requests], own, 74, dtype), [1] * requests, heads, 75)


def with_table(c, change):
    """The output over another table, in the output's type: what a kernel that reads
    other pages would give.  None where the change does not reach the table."""
    table = [list(r) for r in c["table"].tolist()]
    change(table)
    if table == c["table"].tolist():
        return None
    out, _, _ = O.attention(c["query_rope"], c["query"], c["ends"], c["lengths"], i32(table), c["k_rope"], c["kv_cache"], SCALE)
    return out.to(c["kv_cache"].dtype)
