"""The 8-bit latent cache's attention where pages' scales are far apart: pages
of zero rows as the append writes them (scale 2^-126), tiny and huge scales,
and a page that holds a row's maximum at a larger scale than the others."""

from __future__ import annotations

import math

import pytest
import torch

from _latent8 import DTYPES, PAGE, SCALE, i32, make_cache, queries, weights_bound, wide_attention, wide_bound

pytestmark = pytest.mark.gpu


def _api():
    from nanovllm_amd import latent_cache

    return latent_cache


def _attend(c, qr, q, ends, topk=None, weights=True):
    """Outputs and token records of one call against the 64-bit form."""
    batch = len(c["lengths"])
    out = torch.full_like(q, 7.0).cuda()
    entries = torch.arange(batch, dtype=torch.int32)
    records = torch.zeros(batch, c["cols"] * PAGE).cuda() if weights and topk is None else None
    _api().latent8_attention(qr.cuda(), q.cuda(), ends.cuda(), c["lengths"].cuda(), c["table"].cuda(), c["cache"].cuda(),
                             c["scale"].cuda(), SCALE, out, topk_ids=None if topk is None else topk.cuda(),
                             req_pool_entries=None if records is None else entries.cuda(), token_weights=records)
    torch.cuda.synchronize()
    want, sums, size, reach, tail = wide_attention(qr, q, ends, c, topk)
    keys = c["cols"] * PAGE if topk is None else topk.shape[1]
    err = (out.cpu().double() - want).abs()
    bound = wide_bound(want, size, reach, tail, q.dtype, keys)
    assert (err <= bound).all(), f"worst {float((err / bound).nan_to_num(math.inf).max())} of the bound"
    if records is not None:
        terms = int(torch.diff(ends, prepend=i32([0])).max()) * q.shape[1]
        # (2^-13: the exponents' roundings, see wide_bound.)
        off = weights_bound(sums, sums, reach, keys, terms) + sums * 2.0 ** -13
        assert ((records.cpu().double() - sums).abs() <= off).all()


def _appended(lengths, zero, latent_heads, dtype, seed, size=1.0):
    """A cache that latent8_append filled: rows of zeros in the slots that
    ``zero(b, slots)`` names, normal ones elsewhere."""
    c = make_cache(lengths, latent_heads, seed=seed)
    g = torch.Generator().manual_seed(seed)
    kv, rope = torch.randn(sum(lengths), latent_heads, 512, generator=g), torch.randn(sum(lengths), latent_heads, 64, generator=g)
    row = 0
    for b, n in enumerate(lengths):
        blank = zero(b, torch.arange(n)).nonzero().flatten() + row
        kv[blank], rope[blank] = 0, 0
        row += n
    ends = torch.tensor(lengths).cumsum(0).to(torch.int32)
    d = {k: c[k].cuda() for k in ("cache", "scale")}
    _api().latent8_append((kv * size).to(dtype).cuda(), (rope * size).to(dtype).cuda(), ends.cuda(), c["lengths"].cuda(),
                          c["table"].cuda(), d["cache"], d["scale"])
    return {**c, "cache": d["cache"].cpu(), "scale": d["scale"].cpu()}


def _lists(c, rows, width, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-2, int(c["lengths"].min()) + 20, (rows, width), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("lengths", [[1], [4], [128], [300, 4, 1], [5000]])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_requests_of_zero_rows(lengths, dtype):
    """Every key weighs the same: outputs of zero, weights of 1 / n."""
    print(f"ZERO REQUESTS {lengths} {dtype}", flush=True)
    c = _appended(lengths, lambda b, s: s >= 0, 1, DTYPES[dtype], 3)
    assert (c["scale"][c["table"][0, 0]] == 2.0 ** -126).all()
    qr, q, ends = queries([1] * len(lengths), 16, DTYPES[dtype], 3)
    _attend(c, qr, q, ends)
    _attend(c, qr, q, ends, _lists(c, len(lengths), 90, 1))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,latent_heads", [(64, 1), (10, 2)])
def test_first_page_of_zero_rows(heads, latent_heads, dtype):
    print(f"ZERO FIRST {heads} {dtype}", flush=True)
    c = _appended([700, 130], lambda b, s: s < PAGE, latent_heads, DTYPES[dtype], 5)
    for size in (0.1, 2.0, 12.0):
        qr, q, ends = queries([2, 1], heads, DTYPES[dtype], 5, size=size)
        _attend(c, qr, q, ends)
        _attend(c, qr, q, ends, _lists(c, 3, 200, 2))
        _attend(c, qr, q, ends, torch.arange(700, dtype=torch.int32).expand(3, 700).contiguous())


@pytest.mark.parametrize("boost", [0.0, 3.0, 12.0])
def test_pages_of_zero_rows_behind_large_scores(boost):
    """Ordinary pages whose scores lie `boost` above zero on average, zero
    pages (score 0) after and between them."""
    print(f"ZERO LATER {boost}", flush=True)
    c = _appended([900, 515], lambda b, s: (s // PAGE) % 3 != 0, 1, torch.bfloat16, 7)
    c["cache"].view(torch.uint8)[..., 575] = torch.where(c["cache"].float()[..., 575] == 0, 0, 0x7E).to(torch.uint8)  # 448
    qr, q, ends = queries([3, 1], 20, torch.bfloat16, 7, size=0.5)
    qr[..., 63] = boost / (448 * 2.0 ** -6 * SCALE)
    _attend(c, qr, q, ends)
    _attend(c, qr, q, ends, _lists(c, 4, 333, 3))


def test_parts_that_begin_in_zero_pages():
    """One request over every part of the launch, two of three pages zero."""
    print("ZERO PARTS", flush=True)
    c = _appended([20001], lambda b, s: (s // PAGE) % 3 != 2, 1, torch.bfloat16, 9)
    qr, q, ends = queries([2], 8, torch.bfloat16, 9)
    _attend(c, qr, q, ends)
    c = _appended([500] * 60, lambda b, s: (s // PAGE) % 2 == b % 2, 1, torch.bfloat16, 10)
    qr, q, ends = queries([1] * 60, 8, torch.bfloat16, 10)
    _attend(c, qr, q, ends)
    _attend(c, qr, q, ends, _lists(c, 60, 700, 4))


@pytest.mark.parametrize("exponents", [(-126, -119), (-110, -100), (-63, -57), (60, 80), (105, 112), (-126, 40), (-60, 10)])
def test_scales_of_every_magnitude(exponents):
    """Equal and unequal scores at scales of a caller's own.  Scores stay near
    zero, whatever the scale: the queries see rope codes that are zero at all
    scales but the smallest of the range."""
    print(f"SCALES {exponents}", flush=True)
    c = make_cache([700, 260, 9], 1, seed=11, exponents=exponents)
    c["cache"].view(torch.uint8)[..., 512:] = 0
    qr, q, ends = queries([1, 2, 1], 24, torch.bfloat16, 11)
    q.zero_()
    _attend(c, qr, q, ends)
    _attend(c, qr, q, ends, _lists(c, 4, 150, 5))


def _sink(length, where, ratio, lead, seed):
    """Nearly equal keys of positive values at scale 2^-6, and in page `where`,
    whose scale is 2^ratio larger, one key with 2^lead times their weight and
    values in the first 256 dims only."""
    c = make_cache([length], 1, seed=seed, exponents=(-6, -5))
    g = torch.Generator().manual_seed(seed)
    codes = torch.rand(c["cache"].shape, generator=g) * 6 + 1
    codes[..., 512:] = 0
    codes[..., 513] = torch.randn(codes.shape[:-1], generator=g) * 4
    page = int(c["table"][0, where])
    codes[page] = 0
    codes[page, 60, :, :256], codes[page, 60, :, 512] = 3.0, 64.0
    c["cache"] = codes.to(torch.float8_e4m3fn)
    c["scale"][page] = 2.0 ** (ratio - 6)
    heads = 4
    q = torch.zeros(1, heads, 512, dtype=torch.float16)
    qr = torch.zeros(1, heads, 64, dtype=torch.float16)
    qr[..., 0] = lead * math.log(2) / (64 * 2.0 ** (ratio - 6) * SCALE)
    qr[..., 1] = torch.tensor([0.0, 0.3, 0.01, 1.0]) / (4 * 2.0 ** -6 * SCALE)
    return c, qr, q


@pytest.mark.parametrize("ratio,lead", [(10, 14), (12, 14), (8, 14), (12, 6), (0, 14)])
@pytest.mark.parametrize("where", [0, 100, 250])
def test_maximum_in_a_page_of_a_larger_scale(ratio, lead, where):
    print(f"SINK ratio={ratio} lead={lead} where={where}", flush=True)
    c, qr, q = _sink(32600, where, ratio, lead, 13)
    _attend(c, qr, q, i32([1]))
    g = torch.Generator().manual_seed(14)
    topk = torch.randperm(32600, generator=g)[:1500].to(torch.int32)[None].contiguous()
    topk[0, 700] = where * PAGE + 60
    _attend(c, qr, q, i32([1]), topk)


def test_no_tile_is_left_out():
    """Equal scores and small whole values, so that sums are exact: dims that
    only every ninth tile of 64 keys has values in.  Any one tile left out, or
    taken twice, moves some output by more than the bound (checked here)."""
    print("EVERY TILE", flush=True)
    length, heads = 70001, 3
    c = make_cache([length], 1, seed=15, exponents=(0, 1))
    tiles = torch.arange(c["cols"] * 2)
    hot = (tiles[:, None] * 5 + torch.arange(512)) % 9 == 0                        # [tiles, 512]
    values = torch.randint(4, 8, (len(tiles), 64, 512), generator=torch.Generator().manual_seed(15)) * hot[:, None]
    codes = torch.zeros(c["cache"].shape)
    codes[c["table"][0].long(), :, 0, :512] = values.view(-1, PAGE, 512).float()
    c["cache"] = codes.to(torch.float8_e4m3fn)
    values = values.flatten(0, 1)[:length].double()
    want = values.sum(0) / length
    # fp16's half step, and 2^-21 for the quotient and the products with it.
    bound = want * (2.0 ** -11 + 2.0 ** -21)
    for t in range(0, -(-length // 64)):
        part = values[t * 64:(t + 1) * 64]
        for other in ((values.sum(0) - part.sum(0)) / (length - len(part)), (values.sum(0) + part.sum(0)) / (length + len(part))):
            assert ((other - want).abs() > 2 * bound).any(), t
    q = torch.zeros(1, heads, 512, dtype=torch.float16).cuda()
    out = torch.empty_like(q)
    args = [x.cuda() for x in (i32([1]), c["lengths"], c["table"], c["cache"], c["scale"])]
    _api().latent8_attention(q[..., :64].contiguous(), q, *args, SCALE, out)
    assert ((out[0].cpu().double() - want).abs() <= bound).all()
