"""The 8-bit latent cache on the GPU vs the 64-bit oracle: codes, scales,
records and moves bit for bit, attention and its weights within bounds that
follow from the roundings."""

from __future__ import annotations

import pytest
import torch

from _latent8 import (DTYPES, PAGE, SCALE, attention_bound, i32, make_cache, oracle_attention, queries, same_codes,
                      weights_bound)
from oracle import latent8_oracle as O

pytestmark = pytest.mark.gpu


def _api():
    from nanovllm_amd import latent_cache

    return latent_cache


def _gpu(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


# -------------------------------------------------------------------- append
def _append_case(c, counts, latent_heads, dtype, seed, pool, pad=0, fill=None):
    g = torch.Generator().manual_seed(seed)
    total = sum(counts) + pad
    kv = (torch.randn(total, latent_heads, 512, generator=g) * torch.exp2(torch.rand(total, 1, 1, generator=g) * 4 - 2))
    k_rope = torch.randn(total, latent_heads, 64, generator=g)
    kv, k_rope = kv.to(dtype), k_rope.to(dtype)
    if fill is not None:
        fill(kv, k_rope)
    ends = torch.tensor(counts).cumsum(0).to(torch.int32)
    batch = len(counts)
    extra = {}
    if pool:
        extra = {"positions": torch.randint(0, 1 << 20, (total,), generator=g, dtype=torch.int32),
                 "req_pool_entries": torch.randperm(batch + 1, generator=g)[:batch].to(torch.int32),
                 "token_positions": torch.full((batch + 1, c["cols"] * PAGE), -7, dtype=torch.int32),
                 "token_weights": torch.rand(batch + 1, c["cols"] * PAGE, generator=g)}
    return kv, k_rope, ends, extra


def _check_append(c, kv, k_rope, ends, extra):
    d = {k: v.cuda() for k, v in extra.items()}
    cache, scale = c["cache"].cuda(), c["scale"].cuda()
    _api().latent8_append(*_gpu(kv, k_rope, ends, c["lengths"], c["table"]), cache, scale, **d)
    torch.cuda.synchronize()
    e = {k: v.clone() for k, v in extra.items()}
    O.append(kv, k_rope, ends, c["lengths"], c["table"], c["cache"], c["scale"], e.get("positions"),
             e.get("req_pool_entries"), e.get("token_positions"), e.get("token_weights"))
    assert torch.equal(scale.cpu(), c["scale"])
    assert same_codes(cache, c["cache"])
    for k in ("token_positions", "token_weights"):
        if k in e:
            assert torch.equal(d[k].cpu(), e[k]), k


@pytest.mark.parametrize("past,counts,latent_heads,dtype,pool", [
    ([0], [1], 1, "bf16", False),
    ([127, 128, 5, 300], [1, 1, 1, 1], 1, "bf16", True),
    ([1, 126, 0, 64], [3, 5, 0, 70], 2, "f16", True),
    ([0, 90], [129, 256], 3, "bf16", True),
    ([0, 0, 37], [0, 128, 700], 1, "f16", False),
    ([13] * 37, [i % 4 for i in range(37)], 1, "bf16", True),
])
def test_append(past, counts, latent_heads, dtype, pool):
    print(f"APPEND past={past[:4]} counts={counts[:4]} G={latent_heads} {dtype}", flush=True)
    c = make_cache([p + n for p, n in zip(past, counts)], latent_heads, seed=len(past) + latent_heads)
    _check_append(c, *_append_case(c, counts, latent_heads, DTYPES[dtype], 5, pool, pad=3))


def test_append_many_requests():
    """More requests than a workgroup has threads, empty ones among them."""
    counts = [(i * 7) % 3 for i in range(1200)]
    past = [(i * 13) % 140 for i in range(1200)]
    c = make_cache([p + n for p, n in zip(past, counts)], 1, seed=9)
    print("APPEND many", flush=True)
    _check_append(c, *_append_case(c, counts, 1, torch.bfloat16, 6, True, pad=5))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_append_values(dtype):
    """Infinities, NaN, zeros, the type's extremes, and magnitudes on the
    border of a scale."""
    t = DTYPES[dtype]
    info = torch.finfo(t)

    def fill(kv, rope):
        kv[0] = 0.0
        rope[0] = 0.0
        kv[1, 0, 3], kv[1, 0, 4], kv[1, 0, 5] = float("inf"), float("-inf"), float("nan")
        kv[2, 0, 0] = info.max
        kv[3] = info.tiny
        rope[3] = -info.smallest_normal / 64
        kv[4] = 0.5
        kv[4, 0, 7] = 1.75  # 448 * 2^-8: the last that the scale 2^-8 holds
        rope[4] = 0.5
        kv[5] = 0.5
        kv[5, 0, 7] = 1.75 * (1 + info.eps)
        rope[5] = 0.5
        kv[6] = float("nan")
        rope[6] = float("inf")

    c = make_cache([128 * 2 + 1] + [3, 130, 5, 1, 129, 40], 1, seed=2)
    print(f"APPEND values {dtype}", flush=True)
    _check_append(c, *_append_case(c, [1] * 7, 1, t, 8, False, fill=fill))


def test_append_skips_what_names_nothing():
    """Pages outside the cache, slots before 0 or behind the table, pool rows
    outside the pool, ends that run backwards or past the rows."""
    c = make_cache([200, 140, 90, 60], 1, seed=3, cols=2)
    c["table"][0, 1], c["table"][1, 0] = -1, c["blocks"]
    kv, rope, ends, extra = _append_case(c, [80, 20, 95, 10], 1, torch.bfloat16, 4, True)
    c["lengths"] = i32([200, 300, 90, 60])  # request 1 runs past the table, request 2 begins before slot 0
    extra["req_pool_entries"][3] = 99
    print("APPEND skips", flush=True)
    _check_append(c, kv, rope, ends, extra)
    c = make_cache([200, 140, 90, 60], 1, seed=3, cols=2)
    c["lengths"] = i32([-5, 140, 90, 60])
    print("APPEND backwards ends", flush=True)
    _check_append(c, kv, rope, i32([80, 60, 900, 950]), extra)


def test_append_any_scale():
    """Scales that are no powers of two (a caller's own quantiser) stay where
    they suffice and are divided by; zero, NaN and infinite ones are replaced."""
    c = make_cache([40, 41, 42, 43, 44], 1, seed=6)
    for b, s in enumerate([0.037, 0.0, float("nan"), 3.1e-5, 0.9]):
        c["scale"][c["table"][b, 0]] = s
    print("APPEND any scale", flush=True)
    _check_append(c, *_append_case(c, [1] * 5, 1, torch.bfloat16, 7, False))


# ----------------------------------------------------------------- attention
def _run_attention(c, qr, q, ends, topk=None, entries=None, weights=None, out=None):
    d = _gpu(qr, q, ends, c["lengths"], c["table"], c["cache"], c["scale"])
    out = torch.full_like(d[1], 7.0) if out is None else out
    w = None if weights is None else weights.cuda()
    _api().latent8_attention(*d, SCALE, out, topk_ids=None if topk is None else topk.cuda(),
                             req_pool_entries=None if entries is None else entries.cuda(), token_weights=w)
    torch.cuda.synchronize()
    return out.cpu(), None if w is None else w.cpu()


def _check_attention(c, qr, q, ends, topk=None, weights=False, seed=0):
    batch = len(c["lengths"])
    entries = before = None
    if weights:
        g = torch.Generator().manual_seed(seed)
        entries = torch.randperm(batch + 2, generator=g)[:batch].to(torch.int32)
        before = torch.rand(batch + 2, c["cols"] * PAGE, generator=g)
    out, after = _run_attention(c, qr, q, ends, topk, entries, before)
    want, sums, size, reach = oracle_attention(qr, q, ends, c, topk)
    mine = ~want.isnan().any(-1).any(-1)
    assert (out[~mine] == 7.0).all(), "rows of no request are left as they were"
    keys = c["cols"] * PAGE if topk is None else topk.shape[1]
    err = (out.double() - want).abs()[mine]
    bound = attention_bound(want, size, reach, q.dtype, keys, c["scale"])[mine]
    assert (err <= bound).all(), f"worst {float((err / bound).max())} of the bound"
    if weights:
        expect = before.double()
        for b in range(batch):
            expect[int(entries[b])] += sums[b]
        terms = int(torch.diff(ends, prepend=i32([0])).max()) * q.shape[1]
        bound = weights_bound(expect - before, expect, reach, keys, terms)
        assert ((after.double() - expect).abs() <= bound).all()


@pytest.mark.parametrize("lengths,rows,heads,latent_heads,dtype,weights", [
    ([1], [1], 1, 1, "bf16", False),
    ([0], [1], 4, 1, "bf16", True),
    ([63, 64, 65], [1, 1, 1], 16, 1, "bf16", True),
    ([127, 128, 129, 1], [1, 1, 1, 1], 5, 1, "f16", True),
    ([700, 3, 1500], [1, 1, 1], 64, 1, "bf16", False),
    ([333, 2], [1, 1], 65, 1, "f16", True),
    ([200, 1024], [1, 1], 128, 2, "bf16", True),
    ([5, 2, 400, 64], [4, 4, 4, 4], 16, 1, "bf16", True),        # rows that see nothing: 2 cached, 4 rows
    ([300, 77], [65, 13], 6, 3, "f16", True),
    ([257, 0, 130], [257, 3, 0], 8, 2, "bf16", True),            # a whole prompt, an empty one, none
    ([640], [150], 32, 1, "bf16", False),
    ([90] * 5, [1, 0, 2, 3, 1], 40, 1, "f16", True),
])
def test_attention(lengths, rows, heads, latent_heads, dtype, weights):
    print(f"ATTENTION {lengths} rows={rows} N={heads} G={latent_heads} {dtype} w={weights}", flush=True)
    c = make_cache(lengths, latent_heads, seed=sum(lengths) + heads)
    qr, q, ends = queries(rows, heads, DTYPES[dtype], heads, pad=2)
    _check_attention(c, qr, q, ends, weights=weights, seed=heads)


@pytest.mark.parametrize("size,spread", [(0.0, (-7, -6)), (30.0, (-7, -5)), (1.0, (-30, 20))])
def test_attention_scores_and_scales(size, spread):
    """Equal scores; scores of hundreds (one key takes all); pages whose
    scales lie 2^50 apart."""
    c = make_cache([900, 333], 1, seed=11, exponents=spread)
    print(f"ATTENTION size={size} scales={spread}", flush=True)
    if spread[1] > 0:
        # Equal scores, so every page's values count: the queries see only zeros in the rope part.
        c["cache"].view(torch.uint8)[..., 512:] = 0
        qr, q, ends = queries([1, 2], 8, torch.bfloat16, 3, size=size)
        q.zero_()
    else:
        qr, q, ends = queries([1, 2], 8, torch.bfloat16, 3, size=size)
    _check_attention(c, qr, q, ends, weights=True, seed=1)


@pytest.mark.parametrize("lengths,rows,heads,latent_heads,width,dtype", [
    ([300], [1], 4, 1, 1, "bf16"),
    ([1000, 64, 1], [1, 1, 1], 16, 1, 70, "f16"),
    ([900, 1300], [1, 4], 64, 1, 513, "bf16"),
    ([2500], [3], 130, 2, 2048, "bf16"),
    ([400, 400], [2, 2], 8, 1, 1100, "f16"),
])
def test_attention_list(lengths, rows, heads, latent_heads, width, dtype):
    """Lists with entries that name nothing: -1, behind the row's last slot,
    far outside; one list without any valid entry; one slot listed twice."""
    print(f"LIST {lengths} rows={rows} N={heads} K={width}", flush=True)
    c = make_cache(lengths, latent_heads, seed=width)
    qr, q, ends = queries(rows, heads, DTYPES[dtype], width, pad=1)
    g = torch.Generator().manual_seed(width)
    topk = torch.randint(-3, max(lengths) + 40, (q.shape[0], width), generator=g, dtype=torch.int32)
    if width > 3:
        topk[0, 1], topk[0, 2], topk[0, 3] = topk[0, 0], 2 ** 31 - 1, -2 ** 31
    if sum(rows) > 1:
        topk[1] = -1
    _check_attention(c, qr, q, ends, topk=topk)


def test_attention_many_requests():
    """More requests than a workgroup has threads; lengths from none to many."""
    lengths = [(i * 37) % 90 for i in range(700)]
    lengths[640] = 3000
    c = make_cache(lengths, 1, seed=5)
    qr, q, ends = queries([1] * 700, 2, torch.bfloat16, 5)
    print("ATTENTION many", flush=True)
    _check_attention(c, qr, q, ends, weights=True, seed=2)


@pytest.mark.parametrize("topk", [False, True])
def test_attention_many_requests_few_rows(topk):
    """More requests than a workgroup has threads, most of them without rows:
    the few items are split one by one."""
    lengths = [(i * 61) % 700 + 40 for i in range(620)]
    rows = [i % 31 == 3 for i in range(620)]
    lengths = [n if r else 5 for n, r in zip(lengths, rows)]
    c = make_cache(lengths, 1, seed=27)
    qr, q, ends = queries([int(r) for r in rows], 20, torch.bfloat16, 27)
    lists = None
    if topk:
        lists = torch.randint(-1, 60, (q.shape[0], 700), generator=torch.Generator().manual_seed(27), dtype=torch.int32)
    print(f"ATTENTION few rows topk={topk}", flush=True)
    _check_attention(c, qr, q, ends, topk=lists, weights=not topk, seed=7)


def test_attention_long():
    """One request across every part of the launch, window changes among them."""
    c = make_cache([70001, 40], 1, seed=8)
    qr, q, ends = queries([2, 1], 3, torch.bfloat16, 8)
    print("ATTENTION long", flush=True)
    _check_attention(c, qr, q, ends, weights=True, seed=3)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_scales_of_any_size(dtype):
    """Scales that are no powers of two, in dense order and in a list's."""
    c = make_cache([1500, 200], 1, seed=17)
    c["scale"] *= 1 + torch.rand(c["scale"].shape, generator=torch.Generator().manual_seed(17))
    qr, q, ends = queries([2, 1], 24, DTYPES[dtype], 17)
    print(f"ATTENTION scales {dtype}", flush=True)
    _check_attention(c, qr, q, ends, weights=True, seed=5)
    topk = torch.randint(0, 200, (3, 333), generator=torch.Generator().manual_seed(18), dtype=torch.int32)
    _check_attention(c, qr, q, ends, topk=topk)


@pytest.mark.parametrize("heads,step", [(64, 40.0), (64, 12.0), (20, 300.0)])
def test_attention_scores_that_grow(heads, step):
    """Scores that grow from tile to tile by `step` for some rows, fall for
    others and stay for the rest: references follow late and in either group."""
    c = make_cache([832], 1, seed=19)
    sign = torch.where(torch.rand(576, generator=torch.Generator().manual_seed(19)) < 0.5, -1.0, 1.0)
    for page in range(7):
        tile = torch.arange(page * PAGE, (page + 1) * PAGE) // 64
        codes = torch.where(sign > 0, 1.0, -1.0) * (tile.float() * 8 + 1)[:, None]
        c["cache"][int(c["table"][0, page]), :, 0] = codes.to(torch.float8_e4m3fn)
    c["scale"].fill_(2.0 ** -6)
    # 576 * 8 codes a tile at that scale and factor: q of `size` moves a score by `step` a tile.
    size = step / (576 * 8 * 2.0 ** -6 * SCALE)
    way = torch.tensor([1.0, -1.0, 0.0])[torch.arange(heads) % 3]
    both = (sign * size)[None, None] * way[None, :, None]
    q, qr = both[..., :512].contiguous().bfloat16(), both[..., 512:].contiguous().bfloat16()
    print(f"ATTENTION growing N={heads} step={step}", flush=True)
    _check_attention(c, qr, q, i32([1]), weights=True, seed=6)
    topk = torch.arange(832, dtype=torch.int32)[None].contiguous()
    _check_attention(c, qr, q, i32([1]), topk=topk)


def test_attention_many_long_requests():
    """22 requests of 806,000 tokens each in three pages: more tiles a part than
    pages are resolved at a time, more slices than sums are held.  Equal scores
    and small whole values: p is 1, and every sum is exact in fp32 (below 2^24)
    up to the division and the store."""
    cols, length, batch, heads = 6300, 806_000, 22, 64
    g = torch.Generator().manual_seed(20)
    cache = torch.randint(0, 4, (3, PAGE, 1, 576), generator=g).float()
    cache[0, ..., 170:], cache[1, ..., :170], cache[1, ..., 340:], cache[2, ..., :340] = 0, 0, 0, 0
    row = torch.randint(0, 3, (cols,), generator=g, dtype=torch.int32)
    seen = torch.zeros(3, PAGE, dtype=torch.float64)
    for page in range(3):
        at = (row == page).nonzero().flatten() * PAGE
        seen[page] = ((at[:, None] + torch.arange(PAGE)) < length).sum(0)
    want = torch.einsum("pk,pkd->d", seen, cache[:, :, 0, :512].double()) / length
    zero = torch.zeros(batch, heads, 576, dtype=torch.float16)
    c = {"cache": cache.to(torch.float8_e4m3fn), "scale": torch.ones(3, 1), "table": row.expand(batch, cols).contiguous(),
         "lengths": i32([length] * batch)}
    weights = torch.zeros(batch, cols * PAGE)
    print("ATTENTION many long", flush=True)
    out, after = _run_attention(c, zero[..., :64].contiguous(), zero[..., :512].contiguous(),
                                torch.arange(1, batch + 1, dtype=torch.int32), entries=torch.arange(batch, dtype=torch.int32),
                                weights=weights)
    # fp16's half step, and 2^-22 for 1 / l and the product with it.
    assert ((out.double() - want).abs() <= want * (2.0 ** -11 + 2.0 ** -22)).all()
    # p = 2^-lse with lse = log2(806,000) < 32: 2^-20 and the logarithm's and the
    # exponential's 2^-21 each, times ln 2 and once more for the sum of 64.
    assert ((after[:, :length].double() * length / heads - 1).abs() <= 2.0 ** -19).all()
    assert (after[:, length:] == 0).all()


def test_attention_with_ends_that_decrease():
    """More items than the rows can have: nothing is done, to the records
    neither (the workspace holds what another call left there)."""
    c = make_cache([90, 40, 130, 60, 128], 1, seed=29)
    qr, q, _ = queries([130], 1, torch.bfloat16, 29)
    before = torch.rand(5, c["cols"] * PAGE)
    from nanovllm_amd import _lib

    size = _lib.lib.nvdsa_latent8_attention_workspace_size(130, 1, 1)
    torch.cuda.empty_cache()
    torch.zeros(size, dtype=torch.uint8, device="cuda")
    print("ATTENTION decreasing ends", flush=True)
    out, after = _run_attention(c, qr, q, i32([130, 1, 130, 1, 130]), entries=torch.arange(5, dtype=torch.int32),
                                weights=before)
    assert (out == 7.0).all() and torch.equal(after, before)


def test_attention_list_of_many_windows():
    """Parts of a list that are longer than the entries resolved at a time."""
    lengths = [700 - 3 * i for i in range(60)]
    c = make_cache(lengths, 1, seed=21)
    qr, q, ends = queries([1] * 60, 3, torch.bfloat16, 21)
    topk = torch.randint(-1, 720, (60, 8200), generator=torch.Generator().manual_seed(21), dtype=torch.int32)
    print("LIST many windows", flush=True)
    _check_attention(c, qr, q, ends, topk=topk)


def test_attention_nan_in_unseen_places():
    """NaN codes behind the last token, and in tokens that only later rows
    see, leave the rows that do not see them alone; rows that see one are NaN."""
    c = make_cache([200, 130], 1, seed=12)
    codes = c["cache"].view(torch.uint8)
    clean = codes.clone()
    for b, n in enumerate([200, 130]):
        page = int(c["table"][b, n // PAGE])
        codes[page, n % PAGE:] = 0x7F
    unused = sorted(set(range(c["blocks"])) - set(c["table"].flatten().tolist()))
    codes[unused] = 0xFF
    qr, q, ends = queries([4, 1], 16, torch.bfloat16, 12)
    print("ATTENTION NaN", flush=True)
    got, _ = _run_attention(c, qr, q, ends)
    other = {**c, "cache": clean.view(torch.float8_e4m3fn)}
    want, _ = _run_attention(other, qr, q, ends)
    assert torch.equal(got, want) and not got.isnan().any()
    page = int(c["table"][0, 198 // PAGE])
    codes[page, 198 % PAGE] = 0x7F  # seen by the last two of request 0's four rows
    got, _ = _run_attention(c, qr, q, ends)
    assert torch.equal(got[[0, 1, 4]], want[[0, 1, 4]])
    assert got[2:4].isnan().all()
    topk = torch.arange(190, 222, dtype=torch.int32).expand(5, 32).contiguous()
    got, _ = _run_attention(c, qr, q, ends, topk)
    assert not got[[0, 1, 4]].isnan().any() and got[2:4].isnan().all() and (got[4] == 0).all()


def test_attention_pages_that_name_nothing():
    c = make_cache([500, 260], 1, seed=13)
    c["table"][0, 1], c["table"][1, 0], c["table"][1, 1], c["table"][1, 2] = -4, c["blocks"], -1, 2 ** 30
    qr, q, ends = queries([2, 1], 8, torch.bfloat16, 13)
    print("ATTENTION bad pages", flush=True)
    _check_attention(c, qr, q, ends, weights=True, seed=4)
    topk = torch.arange(100, 300, dtype=torch.int32).expand(3, 200).contiguous()
    _check_attention(c, qr, q, ends, topk=topk)
    entries = i32([9, -1])  # pool rows that name nothing: no weights are written
    before = torch.rand(3, c["cols"] * PAGE)
    _, after = _run_attention(c, qr, q, ends, entries=entries, weights=before)
    assert torch.equal(before, after)


def test_attention_offsets_past_32_bits():
    """Pages beyond 4 GiB of cache."""
    blocks = 60_000
    cache = torch.zeros(blocks, PAGE, 1, 576, dtype=torch.uint8, device="cuda")
    c = make_cache([300], 1, seed=14)
    far = torch.tensor([59_999, 58_500, 59_000])
    assert int(far.min()) * PAGE * 576 > 2 ** 32
    cache[far.cuda()] = c["cache"].view(torch.uint8)[c["table"][0].long()].cuda()
    scale = torch.ones(blocks, 1, device="cuda")
    scale[far.cuda()] = c["scale"][c["table"][0].long()].cuda()
    qr, q, ends = queries([1], 8, torch.bfloat16, 14)
    table = far.to(torch.int32)[None].contiguous().cuda()
    out = torch.empty_like(q, device="cuda")
    print("ATTENTION far pages", flush=True)
    args = _gpu(qr, q, ends, c["lengths"])
    _api().latent8_attention(*args, table, cache.view(torch.float8_e4m3fn), scale, SCALE, out)
    want, _ = _run_attention(c, qr, q, ends)
    assert torch.equal(out.cpu(), want)
    kv, rope = torch.randn(1, 1, 512).bfloat16(), torch.randn(1, 1, 64).bfloat16()
    _api().latent8_append(*_gpu(kv, rope, i32([1]), i32([301])), table, cache.view(torch.float8_e4m3fn), scale)
    O.append(kv, rope, i32([1]), i32([301]), c["table"], c["cache"], c["scale"])
    assert same_codes(cache[far.cuda()], c["cache"][c["table"][0].long()])


# ------------------------------------------------------------------ eviction
def _records(c, seed, pool_rows=None, positions=None):
    g = torch.Generator().manual_seed(seed)
    rows = pool_rows or len(c["lengths"]) + 2
    shape = (rows, c["cols"] * PAGE)
    weights = torch.exp(2 * torch.randn(shape, generator=g)) * (torch.rand(shape, generator=g) < 0.8)
    pos = torch.arange(shape[1], dtype=torch.int32).repeat(rows, 1) if positions is None else positions
    entries = torch.randperm(rows, generator=g)[:len(c["lengths"])].to(torch.int32)
    return weights, pos, entries


def _check_evict(c, budgets, weights, positions, entries, first, last):
    batch, cap = len(c["lengths"]), c["cols"] * PAGE
    d = _gpu(c["lengths"], i32(budgets), c["table"], entries, c["cache"], c["scale"], positions, weights)
    src, dst = torch.full((batch, cap), -9, dtype=torch.int32).cuda(), torch.full((batch, cap), -9, dtype=torch.int32).cuda()
    counts, kept = torch.full((batch,), -9, dtype=torch.int32).cuda(), torch.full((batch,), -9, dtype=torch.int32).cuda()
    _api().latent8_evict(*d, src, dst, counts, kept, protect_first=first, protect_last=last)
    torch.cuda.synchronize()
    moves, lengths = O.evict(c["lengths"], i32(budgets), c["table"], entries, c["cache"], c["scale"], positions, weights,
                             first, last)
    assert kept.tolist() == lengths
    assert counts.tolist() == [len(m) for m in moves]
    for b, m in enumerate(moves):
        assert src[b, :len(m)].tolist() == [s for s, _ in m]
        assert dst[b, :len(m)].tolist() == [h for _, h in m]
        assert (src[b, len(m):] == -9).all() and (dst[b, len(m):] == -9).all()
    assert torch.equal(d[5].cpu(), c["scale"])
    assert same_codes(d[4], c["cache"])
    assert torch.equal(d[6].cpu(), positions)
    assert torch.equal(d[7].cpu().view(torch.int32), weights.view(torch.int32))
    return lengths


@pytest.mark.parametrize("lengths,budgets,latent_heads,first,last", [
    ([130], [128], 1, 0, 1),
    ([300], [1], 1, 0, 0),
    ([129, 128, 127, 1, 0], [100, 128, 200, 0, 5], 1, 4, 16),
    ([700, 1000, 513], [512, 999, 300], 2, 4, 64),
    ([2176, 1500], [2048, 700], 1, 64, 128),
    ([400, 400], [100, -3], 3, 90, 90),          # more protected tokens than the budget; a negative budget
    ([5000], [4097], 1, 4, 128),
])
def test_evict(lengths, budgets, latent_heads, first, last):
    print(f"EVICT {lengths} -> {budgets} G={latent_heads}", flush=True)
    c = make_cache(lengths, latent_heads, seed=sum(lengths), exponents=(-9, -4))
    weights, positions, entries = _records(c, sum(budgets))
    _check_evict(c, budgets, weights, positions, entries, first, last)


def test_evict_ties_and_odd_weights():
    """Equal weights go to the lower slot; -0 is 0; NaN counts above all."""
    c = make_cache([600, 600, 600], 1, seed=21)
    weights, positions, entries = _records(c, 3)
    e = entries.long()
    weights[e[0]] = 1.0
    weights[e[1]] = torch.where(torch.arange(weights.shape[1]) % 3 == 0, -0.0, 0.0)
    weights[e[2], 100:140] = float("nan")
    weights[e[2], 500:510] = float("inf")
    weights[e[2], 300:310] = -1.0
    print("EVICT ties", flush=True)
    _check_evict(c, [333, 200, 45], weights, positions, entries, 2, 5)


def test_evict_nan_of_either_sign():
    c = make_cache([500], 1, seed=25)
    weights, positions, entries = _records(c, 7)
    row = weights[entries.long()[0]].view(torch.int32)
    row[100:130], row[130:150], row[480:490] = -1, -0x400000, 0x7f800001  # NaN: of all ones, negative, signalling
    print("EVICT NaN", flush=True)
    _check_evict(c, [70], weights, positions, entries, 2, 5)


@pytest.mark.parametrize("lengths,budgets", [([32769, 8193], [32640, 4000]), ([40001], [17000])])
def test_evict_long(lengths, budgets):
    """More slots than a workgroup holds in registers."""
    print(f"EVICT long {lengths} -> {budgets}", flush=True)
    c = make_cache(lengths, 1, seed=26)
    weights, positions, entries = _records(c, 8)
    weights[:, 1000:3000] = 0.25  # more equal weights than the budget leaves room for, or none
    _check_evict(c, budgets, weights, positions, entries, 64, 500)


def test_evict_positions_in_any_order():
    """Protection goes by position, not by slot: what an earlier eviction left."""
    c = make_cache([900, 300], 1, seed=22)
    g = torch.Generator().manual_seed(1)
    positions = torch.stack([torch.randperm(c["cols"] * PAGE, generator=g).to(torch.int32) for _ in range(4)])
    weights, positions, entries = _records(c, 4, pool_rows=4, positions=positions)
    print("EVICT positions", flush=True)
    _check_evict(c, [700, 200], weights, positions, entries, 30, 200)


def test_evict_skips_what_names_nothing():
    """Pool rows outside the pool leave a request alone; moves from or to pages
    outside the cache carry the records only."""
    c = make_cache([700, 700], 1, seed=23)
    weights, positions, entries = _records(c, 5)
    entries[1] = 77
    c["table"][0, 1], c["table"][0, 5] = -1, c["blocks"] + 3
    print("EVICT skips", flush=True)
    _check_evict(c, [500, 500], weights, positions, entries, 0, 0)


def test_evict_keeps_lengths_in_place():
    c = make_cache([300, 90], 1, seed=24)
    weights, positions, entries = _records(c, 6)
    d = _gpu(c["lengths"], i32([200, 200]), c["table"], entries, c["cache"], c["scale"], positions, weights)
    lists = [torch.empty(2, c["cols"] * PAGE, dtype=torch.int32, device="cuda") for _ in range(2)]
    print("EVICT in place", flush=True)
    _api().latent8_evict(*d, *lists, torch.empty(2, dtype=torch.int32, device="cuda"), d[0])
    assert d[0].tolist() == [200, 90]


def test_registered_operators_are_the_same():
    """By name, as a traced program calls them: the same outputs."""
    c = make_cache([300, 140], 1, seed=28)
    qr, q, ends = queries([1, 2], 8, torch.bfloat16, 28)
    weights, positions, entries = _records(c, 9)
    print("BY NAME", flush=True)
    state = []
    for by_name in (False, True):
        ops = torch.ops.nanovllm_dsa
        d = dict(zip(("qr", "q", "ends", "lens", "table", "cache", "scale", "entries", "pos", "w"),
                     _gpu(qr, q, ends, c["lengths"], c["table"], c["cache"].clone(), c["scale"].clone(), entries,
                          positions.clone(), weights.clone())))
        out, kv = torch.zeros_like(d["q"]), d["q"][:, :1].contiguous()
        rope = d["qr"][:, :1].contiguous()
        lists = [torch.zeros(2, c["cols"] * PAGE, dtype=torch.int32, device="cuda") for _ in range(2)]
        counts, kept = (torch.zeros(2, dtype=torch.int32, device="cuda") for _ in range(2))
        budgets = i32([200, 128]).cuda()
        if by_name:
            ops.latent8_append(kv, rope, d["ends"], d["lens"], d["table"], d["cache"], d["scale"])
            ops.latent8_attention(d["qr"], d["q"], d["ends"], d["lens"], d["table"], d["cache"], d["scale"], SCALE, out,
                                  None, d["entries"], d["w"])
            ops.latent8_evict(d["lens"], budgets, d["table"], d["entries"], d["cache"], d["scale"], d["pos"], d["w"],
                              *lists, counts, kept, 2, 9)
        else:
            _api().latent8_append(kv, rope, d["ends"], d["lens"], d["table"], d["cache"], d["scale"])
            _api().latent8_attention(d["qr"], d["q"], d["ends"], d["lens"], d["table"], d["cache"], d["scale"], SCALE, out,
                                     req_pool_entries=d["entries"], token_weights=d["w"])
            _api().latent8_evict(d["lens"], budgets, d["table"], d["entries"], d["cache"], d["scale"], d["pos"], d["w"],
                                 *lists, counts, kept, protect_first=2, protect_last=9)
        state.append([out, d["cache"].view(torch.uint8), d["scale"], d["pos"], d["w"], *lists, counts, kept])
    for mine, named in zip(*state):
        assert torch.equal(mine, named)


# ------------------------------------------------------- the three together
def _chain(steps, dtype, latent_heads, heads, seed):
    """Prompts, then decode steps that append, attend with weights, and evict
    requests over their budget; every state checked against the oracle."""
    lengths, budgets = [150, 260, 30], [140, 256, 200]
    c = make_cache([400, 400, 400], latent_heads, seed=seed)
    batch = 3
    g = torch.Generator().manual_seed(seed)
    entries = i32([2, 0, 3])
    positions = torch.zeros(4, c["cols"] * PAGE, dtype=torch.int32)
    weights = torch.zeros(4, c["cols"] * PAGE)
    dev = {k: v.cuda() for k, v in {"cache": c["cache"], "scale": c["scale"], "table": c["table"], "entries": entries,
                                    "positions": positions, "weights": weights}.items()}
    api = _api()
    have, nxt = [0] * batch, [0] * batch
    for step in range(steps):
        counts = lengths if step == 0 else [1, 2, 1]
        total = sum(counts)
        kv = torch.randn(total, latent_heads, 512, generator=g).to(dtype)
        rope = torch.randn(total, latent_heads, 64, generator=g).to(dtype)
        qr, q, ends = queries(counts, heads, dtype, seed + step)
        row_pos = torch.cat([torch.arange(nxt[b], nxt[b] + n) for b, n in enumerate(counts)]).to(torch.int32)
        have = [h + n for h, n in zip(have, counts)]
        nxt = [p + n for p, n in zip(nxt, counts)]
        now = i32(have)
        records = dict(req_pool_entries=dev["entries"], token_weights=dev["weights"])
        ends_g, now_g = ends.cuda(), now.cuda()
        api.latent8_append(kv.cuda(), rope.cuda(), ends_g, now_g, dev["table"], dev["cache"], dev["scale"],
                           positions=row_pos.cuda(), token_positions=dev["positions"], **records)
        O.append(kv, rope, ends, now, c["table"], c["cache"], c["scale"], row_pos, entries, positions, weights)
        assert same_codes(dev["cache"], c["cache"]) and torch.equal(dev["scale"].cpu(), c["scale"])
        assert torch.equal(dev["positions"].cpu(), positions)
        out = torch.empty_like(q).cuda()
        api.latent8_attention(qr.cuda(), q.cuda(), ends_g, now_g, dev["table"], dev["cache"], dev["scale"], SCALE, out,
                              **records)
        want, sums, size, reach = O.attention(qr, q, ends, now, c["table"], c["cache"], c["scale"], SCALE)
        bound = attention_bound(want, size, reach, dtype, c["cols"] * PAGE, c["scale"])
        assert ((out.cpu().double() - want).abs() <= bound).all()
        total = weights.double()
        for b in range(batch):
            total[int(entries[b])] += sums[b]
        bound = weights_bound(total - weights, total, reach, c["cols"] * PAGE, max(counts) * heads)
        assert ((dev["weights"].cpu().double() - total).abs() <= bound).all()
        weights.copy_(dev["weights"].cpu())  # (the selection below goes by these)
        lists = [torch.empty(batch, c["cols"] * PAGE, dtype=torch.int32, device="cuda") for _ in range(2)]
        counts_g, kept = (torch.empty(batch, dtype=torch.int32, device="cuda") for _ in range(2))
        api.latent8_evict(now_g, i32(budgets).cuda(), dev["table"], dev["entries"], dev["cache"], dev["scale"],
                          dev["positions"], dev["weights"], *lists, counts_g, kept, protect_first=2, protect_last=16)
        _, have = O.evict(now, i32(budgets), c["table"], entries, c["cache"], c["scale"], positions, weights, 2, 16)
        assert kept.tolist() == have
        assert same_codes(dev["cache"], c["cache"]) and torch.equal(dev["scale"].cpu(), c["scale"])
        assert torch.equal(dev["positions"].cpu(), positions) and torch.equal(dev["weights"].cpu(), weights)


@pytest.mark.parametrize("dtype,latent_heads,heads", [("bf16", 1, 16), ("f16", 2, 6)])
def test_chain(dtype, latent_heads, heads):
    print(f"CHAIN {dtype} G={latent_heads}", flush=True)
    _chain(5, DTYPES[dtype], latent_heads, heads, 31)


def test_graphs_and_streams():
    """Two captured decode steps (append, attention with weights, eviction) on
    streams of their own, replayed in turn with eager work between: each
    replay gives what the same calls give eagerly."""
    api = _api()
    steps = []
    for seed in (41, 42):
        c = make_cache([500, 300, 900], 1, seed=seed)
        weights, positions, entries = _records(c, seed)
        qr, q, ends = queries([1, 1, 1], 32, torch.bfloat16, seed)
        g = torch.Generator().manual_seed(seed)
        kv, rope = torch.randn(3, 1, 512, generator=g).bfloat16(), torch.randn(3, 1, 64, generator=g).bfloat16()
        t = dict(zip(("qr", "q", "ends", "len", "table", "cache", "scale", "entries", "kv", "rope", "weights", "positions"),
                     _gpu(qr, q, ends, c["lengths"], c["table"], c["cache"], c["scale"], entries, kv, rope, weights,
                          positions)))
        t["row_pos"], t["budgets"] = i32([499, 299, 899]).cuda(), i32([400, 290, 640]).cuda()
        t["out"] = torch.zeros_like(t["q"])
        t["src"], t["dst"] = (torch.zeros(3, c["cols"] * PAGE, dtype=torch.int32, device="cuda") for _ in range(2))
        t["counts"], t["kept"] = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2))
        steps.append(t)
    changed = ("cache", "scale", "weights", "positions", "out", "src", "dst", "counts", "kept")

    def call(t):
        api.latent8_append(t["kv"], t["rope"], t["ends"], t["len"], t["table"], t["cache"], t["scale"],
                           positions=t["row_pos"], req_pool_entries=t["entries"], token_positions=t["positions"],
                           token_weights=t["weights"])
        api.latent8_attention(t["qr"], t["q"], t["ends"], t["len"], t["table"], t["cache"], t["scale"], SCALE, t["out"],
                              req_pool_entries=t["entries"], token_weights=t["weights"])
        api.latent8_evict(t["len"], t["budgets"], t["table"], t["entries"], t["cache"], t["scale"], t["positions"],
                          t["weights"], t["src"], t["dst"], t["counts"], t["kept"], protect_first=4, protect_last=8)

    def restore(t, saved):
        for k in changed:
            t[k].view(torch.uint8).copy_(saved[k].view(torch.uint8))

    print("GRAPHS capture", flush=True)
    graphs, saves, wants = [], [], []
    for t in steps:
        saved = {k: t[k].clone() for k in changed}
        call(t)
        torch.cuda.synchronize()
        wants.append({k: t[k].clone() for k in changed})
        restore(t, saved)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(t)
        restore(t, saved)
        graphs.append(graph)
        saves.append(saved)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for turn in range(4):
        print(f"GRAPHS replay {turn}", flush=True)
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for t, saved, want in zip(steps, saves, wants):
            for k in changed:
                assert torch.equal(t[k].view(torch.uint8), want[k].view(torch.uint8)), (turn, k)
            restore(t, saved)
        eager = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in steps[0].items()}
        with torch.cuda.stream(streams[1]):
            streams[1].wait_stream(torch.cuda.default_stream())
            call(eager)
        torch.cuda.synchronize()
        for k in changed:
            assert torch.equal(eager[k].view(torch.uint8), wants[0][k].view(torch.uint8)), (turn, k, "eager")
