"""The paged cache's operators on the GPU against 64 bits: attention over pages, the weight of pages, appended rows, sealed pages, eviction, and a run of
them together.  The bounds are the arithmetic's, see `paged_cases`."""
import math
import random

import pytest
import torch

from paged_cases import F64, PAGE, Cache, dequantized, evicted
from polarquant_amd.paged import PageBatch, PagePool, evict_pages, page_weights, paged_attention, paged_workspace_bytes, qk_norm_rope_append, seal_pages
from polarquant_amd.quantize import quantize_and_pack_nbit

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def near(got, want, bound, rows=None):
    got = got.to(F64)
    if rows is not None:
        got, want, bound = got[:rows], want[:rows], bound[:rows]
    same = got == want                                  # (infinities)
    off = torch.where(same, 0.0, (got - want).abs() - bound)
    assert bool((off <= 0).all()), "off by %g beyond the bound at %s" % (float(off.max()), torch.nonzero(~(off <= 0))[:3].tolist())


def check_attention(c, scale=None, gone=(), **kw):
    out, lse = paged_attention(c.q, c.pool, kw.pop("batch", c.batch), attention_mask=c.mask, sm_scale=scale, return_lse=True, **kw)
    want, bound, want_lse, lse_bound = c.attention(scale, gone)
    n = sum(c.new)
    near(out, want, bound, n)
    near(lse, want_lse, lse_bound, n)
    return out, lse


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,Nk", [(1, 1), (8, 8), (4, 1), (7, 1), (14, 2), (32, 8), (17, 1), (40, 1)])
def test_attention_of_one_token_and_of_chunks(gpu, dtype, N, Nk):
    """Sequences of one token, none, an end of a page, one behind it, several pages; chunks of one and many tokens, the whole of a sequence."""
    kv = [1, 128, 129, 300, 640, 515, 0, 77]
    new = [1, 1, 1, 5, 33, 130, 0, 77]
    sealed = [0, 0, 1, 2, 4, 3, 0, 0]
    check_attention(Cache(gpu, kv, new, sealed, N, Nk, dtype, seed=N))
    check_attention(Cache(gpu, kv, [min(1, n) for n in kv], [0 if n == 0 else (n - 1) // PAGE for n in kv], N, Nk, dtype, seed=N + 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rbits,tbits,packed", [(1, 1, False), (4, 4, False), (3, 3, False), (3, 3, True), (2, 3, True), (4, 3, False), (5, 2, False), (3, 5, False),
                                                (2, 6, False), (1, 7, False)])
def test_attention_over_codes_of_any_width(gpu, dtype, rbits, tbits, packed):
    for new in ([1, 1], [9, 61]):
        check_attention(Cache(gpu, [401, 260], new, [3, 1], 8, 2, dtype, rbits, tbits, packed, seed=tbits))


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 7, 1]])
def test_attention_masks(gpu, new):
    """Left padding, scattered keys, a sequence of which nothing is seen; the rows behind a mask hold NaN and infinities."""
    c = Cache(gpu, [500, 333, 200], new, [3, 1, 1], 8, 2, torch.bfloat16)
    mask = torch.ones(3, 512, dtype=torch.uint8, device=gpu)
    mask[0, :290] = 0
    mask[1] = (torch.rand(512, generator=torch.Generator(device=gpu).manual_seed(1), device=gpu) < 0.4)
    mask[1, 200:260] = 0
    mask[2] = 0
    c.mask = mask
    for b in range(2):
        for j in range(c.kv[b]):
            if not mask[b, j]:
                c.pool.values[c.pages[b, j // PAGE].item(), :, j % PAGE] = float("nan") if j % 2 else float("inf")
                if j >= c.sealed[b] * PAGE:
                    c.pool.keys[c.open_pages[b, j // PAGE - c.sealed[b]].item(), :, j % PAGE] = float("nan") if j % 2 else float("-inf")
    out, lse = check_attention(c)
    last = slice(int(c.q_start[2]), int(c.q_start[3]))
    assert bool((out[last] == 0).all()) and bool((lse[last] == -math.inf).all())
    for other in (mask.bool(), mask.int() * 3):         # other types count as what is not zero
        assert torch.equal(paged_attention(c.q, c.pool, c.batch, attention_mask=other), out)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 1, 3, 2], [200, 7, 9, 1]])
@pytest.mark.parametrize("units", [None, 0, 64])
def test_attention_behind_long_left_padding(gpu, units, new):
    """Padding over many pages, to the last key, from a page's middle, and of everything; what lies under it is not a number."""
    c = Cache(gpu, [4300, 2049, 3000, 1500], new, [30, 16, 22, 11], 8, 2, torch.float16, seed=7)
    c.mask = torch.ones(4, 4352, dtype=torch.uint8, device=gpu)
    for b, n in enumerate([2500, 2048, 1100, 1500]):
        c.mask[b, :n] = 0
        for j in range(n // PAGE):
            c.pool.values[c.pages[b, j].item()] = float("nan")
    out, _ = check_attention(c, units=units)
    assert bool((out[c.q_start[3]:] == 0).all())


@pytest.mark.parametrize("new", [[1, 1], [50, 3]])
def test_attention_passes_over_pages_that_do_not_exist(gpu, new):
    c = Cache(gpu, [700, 400], new, [4, 2], 8, 2, torch.float16)
    pages, open_pages = c.pages.clone(), c.open_pages.clone()
    pages[0, 1], pages[0, 5], open_pages[1, 0] = -1, 1 << 30, -7
    check_attention(c, gone=[(0, 1), (0, 5), (1, 2)], batch=c.batch_of(pages, open_pages))
    values = c.pages.clone()
    values[0, 2], values[1, 3] = -1, 100000
    check_attention(c, gone=[(0, 2), (1, 3)], batch=c.batch_of(value_pages=values))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0, 0.002])
@pytest.mark.parametrize("new", [[1], [20]])
def test_attention_of_any_scale(gpu, scale, new):
    check_attention(Cache(gpu, [450], new, [2], 8, 2, torch.bfloat16, key_scale=0.5), scale=scale)


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e17), (torch.bfloat16, 1e-17), (torch.float16, 3000.0), (torch.float16, 1e-4)])
def test_attention_of_keys_of_any_size(gpu, dtype, size):
    """Radii are scaled into float16's range page by page, bfloat16 queries row by row.  (The quantizer's radius is the root of a float32 sum of squares: infinite
    from 1.8e19 on, zero below 1e-23, whatever reads it.)"""
    c = Cache(gpu, [450, 300], [1, 30], [3, 1], 8, 2, dtype, key_scale=size)
    c.q[::2] *= 100.0
    check_attention(c, scale=128 ** -0.5 / size / 10)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 5]])
@pytest.mark.parametrize("units", [0, 3, 5, 6, 7, 16, 200])
def test_attention_in_slices(gpu, units, new):
    """However the pages are dealt out; workgroups that get no page; a workspace of the caller's."""
    c = Cache(gpu, [900, 130, 5], new, [6, 0, 0], 8, 2, torch.float16)
    if units == 3 and new[0] > 1:                       # (two row tiles of the first sequence)
        c.new[0] = 30
        c = Cache(gpu, [900, 130, 5], c.new, [6, 0, 0], 8, 2, torch.float16)
    check_attention(c, units=units)
    ws = torch.full((paged_workspace_bytes(c.batch, c.N, c.Nk, units) // 4,), float("nan"), device=gpu)
    check_attention(c, units=units, workspace=ws)


@pytest.mark.parametrize("B", [3, 70, 130])
def test_attention_of_many_sequences_dealt_out(gpu, B):
    """More sequences than a wavefront has lanes, most of a page, some without new tokens, one long."""
    r = random.Random(B)
    kv = [r.randint(1, 200) for _ in range(B)]
    kv[B // 2] = 3000
    new = [r.choice([0, 1, 1, 2]) for _ in range(B)]
    new[B // 2] = 1
    new = [min(n, k) for n, k in zip(new, kv)]
    for units in (2 * B, 2 * B + 17):
        check_attention(Cache(gpu, kv, new, [(k - 1) // PAGE if k > 128 else 0 for k in kv], 4, 1, torch.bfloat16, seed=B), units=units)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rbits,tbits,packed,N,Nk", [(4, 4, False, 8, 2), (3, 3, True, 14, 2), (3, 5, False, 8, 8)])
@pytest.mark.parametrize("units,masked", [(None, False), (0, True), (80, True), (200, False)])
def test_attention_of_batches_that_may_be_long(gpu, dtype, rbits, tbits, packed, N, Nk, units, masked):
    """Of many new tokens and up to 4200 in all: rows in the largest tiles, also for the short sequences of the batch."""
    kv, new = [1, 128, 640, 515, 0, 900, 77, 300], [1, 1, 33, 130, 0, 300, 77, 0]
    c = Cache(gpu, kv, new, [0, 0, 4, 3, 0, 4, 0, 2], N, Nk, dtype, rbits, tbits, packed, seed=N, wide=25)
    b = c.batch
    c.batch = PageBatch(b.q_start, b.kv_len, b.n_sealed, b.pages, b.open_pages, b.max_q, 4200)
    if masked:
        c.mask = (torch.rand(8, 4200, generator=torch.Generator(device=gpu).manual_seed(2), device=gpu) < 0.6).to(torch.uint8)
        c.mask[5, :300] = 0
    check_attention(c, batch=c.batch, units=units)


def test_attention_reads_rows_as_they_lie_and_writes_no_others(gpu):
    """Queries that are a slice of a projection's output; rows of no sequence; tables wider than what is held."""
    c = Cache(gpu, [300, 200], [3, 2], [1, 0], 4, 2, torch.bfloat16, extra_rows=4, wide=3)
    whole = torch.full((c.T, 4 * 128 + 64), float("nan"), dtype=c.dtype, device=gpu)
    whole[:, 32:32 + 512] = c.q.flatten(1)
    c.q = whole[:, 32:32 + 512].unflatten(1, (4, 128))
    out = torch.full((c.T, 4, 128), 7.0, dtype=c.dtype, device=gpu)
    got, _ = check_attention(c, out=out)
    assert got is out and bool((out[5:] == 7.0).all())


@pytest.mark.parametrize("Nk,max_q,units", [(1, 3, 0), (1, 3, 5), (2, 20, 0), (2, 20, 40)])
def test_more_new_tokens_than_max_q_are_cut(gpu, Nk, max_q, units):
    """The first max_q rows of a sequence are its call's; the others are neither read nor written."""
    c = Cache(gpu, [300, 200], [40, 2], [1, 0], 4, Nk, torch.bfloat16)
    b = c.batch
    few = PageBatch(b.q_start, b.kv_len, b.n_sealed, b.pages, b.open_pages, max_q, 300)
    out = torch.full((c.T, 4, 128), 7.0, dtype=c.dtype, device=gpu)
    q = c.q.clone()
    q[max_q:40] = float("nan")
    got, lse = paged_attention(q, c.pool, few, return_lse=True, units=units, out=out)
    rows = list(range(max_q)) + [40, 41]
    packed = PageBatch(torch.tensor([0, max_q, max_q + 2], dtype=torch.int32, device=gpu), b.kv_len, b.n_sealed, b.pages, b.open_pages, max_q, 300)
    want, want_lse = paged_attention(c.q[rows].contiguous(), c.pool, packed, return_lse=True, units=units)
    assert torch.equal(got[rows], want) and torch.equal(lse[rows], want_lse) and bool((out[max_q:40] == 7.0).all())
    lse[max_q:40] = float("nan")
    assert torch.equal(page_weights(q, lse, c.pool, few), page_weights(c.q[rows].contiguous(), want_lse, c.pool, packed))


def test_attention_of_longer_contexts(gpu):
    """Many pages, so that every wavefront goes from page to page and the slices are dealt out unevenly."""
    c = Cache(gpu, [9000, 700, 4111], [1, 1, 1], [70, 5, 32], 28, 4, torch.bfloat16)
    check_attention(c)
    c = Cache(gpu, [5003], [261], [37], 8, 2, torch.float16)
    check_attention(c)


# ---------------------------------------------------------------- weights
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,Nk,rbits,tbits,packed", [(4, 1, 4, 4, False), (14, 2, 3, 3, True), (8, 8, 4, 3, False), (40, 1, 1, 7, False), (70, 1, 4, 4, False)])
def test_page_weights(gpu, dtype, N, Nk, rbits, tbits, packed):
    c = Cache(gpu, [1, 128, 300, 700, 0, 515], [1, 1, 33, 200, 0, 5], [0, 1, 1, 4, 0, 4], N, Nk, dtype, rbits, tbits, packed, wide=2)
    lse = c.attention()[2].float()
    want, bound = c.page_weights(lse, c.pages.shape[1])
    got = page_weights(c.q, lse, c.pool, c.batch)
    near(got, want, bound)
    onto = torch.rand_like(got)
    again = page_weights(c.q, lse, c.pool, c.batch, onto=onto)
    assert torch.equal(again, onto + got)
    near(got.sum((1, 2)), torch.tensor([float(n) * N for n in c.new], dtype=F64, device=gpu), torch.full((6,), 0.02 * N * 200, dtype=F64, device=gpu))


def test_page_weights_behind_a_mask(gpu):
    c = Cache(gpu, [400, 300], [30, 4], [2, 1], 8, 2, torch.bfloat16)
    c.mask = torch.ones(2, 400, dtype=torch.uint8, device=gpu)
    c.mask[0, :200] = 0
    c.mask[1] = 0
    lse = c.attention()[2].float()
    assert bool((lse[30:] == -math.inf).all())
    got = page_weights(c.q, lse, c.pool, c.batch, attention_mask=c.mask)
    want, bound = c.page_weights(lse, c.pages.shape[1])
    near(got, want, bound)
    assert bool((got[1] == 0).all()) and bool((got[0, :, 0] == 0).all())


# ---------------------------------------------------------------- rows
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,Nk,normed", [(32, 8, True), (28, 4, False), (1, 1, True), (6, 3, True)])
def test_append(gpu, dtype, N, Nk, normed):
    """Every row where it belongs and nowhere else.  A row is rounded once, behind float32 sums of two products: u of the result and 8 2^-24 of both products
    (norm, weight, angle)."""
    c = Cache(gpu, [1, 128, 129, 300, 515, 0], [1, 1, 1, 45, 200, 0], [0, 0, 1, 1, 2, 0], N, Nk, dtype, extra_rows=3)
    g = torch.Generator(device=gpu).manual_seed(5)
    qkv = torch.randn(c.T, (N + 2 * Nk) * 128 + 8, generator=g, device=gpu).mul_(3).to(dtype)
    q, k, v = qkv[:, :N * 128], qkv[:, N * 128:(N + Nk) * 128], qkv[:, (N + Nk) * 128:(N + 2 * Nk) * 128]
    angle = torch.rand(600, 128, generator=g, device=gpu) * 6.3
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    w = [torch.randn(128, generator=g, device=gpu).to(dtype) if normed else None for _ in range(2)]
    for positions in (None, torch.randint(-5, 650, (c.T,), generator=g, device=gpu, dtype=torch.int32)):
        c.pool.keys.fill_(7.0)
        c.pool.values.fill_(7.0)
        out = torch.full((c.T, N, 128), 7.0, dtype=dtype, device=gpu)
        got = qk_norm_rope_append(q, k, v, cos, sin, c.pool, c.batch, q_norm=w[0], k_norm=w[1], eps=1e-5, positions=positions, out=out)
        assert got is out
        keys, values = torch.full_like(c.pool.keys, 7.0, dtype=F64), torch.full_like(c.pool.values, 7.0)
        key_bound = torch.zeros_like(keys)
        want, bound = torch.full(out.shape, 7.0, dtype=F64, device=gpu), torch.zeros(out.shape, dtype=F64, device=gpu)
        u = torch.finfo(dtype).eps / 2
        for b, n in enumerate(c.new):
            for t in range(n):
                row, at = int(c.q_start[b]) + t, c.kv[b] - n + t
                a = min(max(at if positions is None else int(positions[row]), 0), 599)
                co, si = cos[a].to(F64), sin[a].to(F64)

                def turned(x, weight):
                    x = x.to(F64).unflatten(-1, (-1, 128))
                    if weight is not None:
                        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * weight.to(F64)
                    other = torch.cat([-x[..., 64:], x[..., :64]], -1)
                    y = x * co + other * si
                    return y, u * y.abs() * (1 + 1e-3) + 8 * 2.0 ** -24 * ((x * co).abs() + (other * si).abs()) + 2.0 ** -25
                want[row], bound[row] = turned(q[row], w[0])
                p = at // PAGE
                if p >= c.sealed[b]:
                    to = c.open_pages[b, p - c.sealed[b]].item()
                    keys[to, :, at % PAGE], key_bound[to, :, at % PAGE] = turned(k[row], w[1])
                values[c.pages[b, p].item(), :, at % PAGE] = v[row].unflatten(-1, (Nk, 128))
        near(out, want, bound)
        near(c.pool.keys, keys, key_bound)
        assert torch.equal(c.pool.values, values)


def test_append_without_a_page(gpu):
    """Rows whose pages do not exist go nowhere, the others to theirs."""
    c = Cache(gpu, [260, 130], [10, 3], [1, 0], 4, 2, torch.float16)
    rows = torch.randn(c.T, 8 * 128, device=gpu).half()
    cos, sin = torch.ones(300, 128, device=gpu).half(), torch.zeros(300, 128, device=gpu).half()
    open_pages, values = c.open_pages.clone(), c.pages.clone()
    open_pages[0, 1], values[1, 0], values[0, 1] = -1, 1 << 20, -1
    c.pool.keys.fill_(7.0)
    c.pool.values.fill_(7.0)
    out = qk_norm_rope_append(rows[:, :512], rows[:, 512:768], rows[:, 768:], cos, sin, c.pool, c.batch_of(open_pages=open_pages, value_pages=values))
    assert torch.equal(out.flatten(1), rows[:, :512])
    keys, vals = torch.full_like(c.pool.keys, 7.0), torch.full_like(c.pool.values, 7.0)
    for t in range(6):                                  # tokens 250 .. 255 of the first sequence: keys; 256 .. 259: values
        keys[c.open_pages[0, 0].item(), :, 122 + t] = rows[t, 512:768].unflatten(0, (2, 128))
    for t in range(6, 10):
        vals[c.pages[0, 2].item(), :, t - 6] = rows[t, 768:].unflatten(0, (2, 128))
    for t in range(10, 13):                             # tokens 127 .. 129 of the second
        at = 127 + t - 10
        keys[c.open_pages[1, at // PAGE].item(), :, at % PAGE] = rows[t, 512:768].unflatten(0, (2, 128))
        if at >= PAGE:
            vals[c.pages[1, 1].item(), :, at % PAGE] = rows[t, 768:].unflatten(0, (2, 128))
    assert torch.equal(c.pool.keys, keys) and torch.equal(c.pool.values, vals)


# ---------------------------------------------------------------- sealing
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rbits,tbits,packed,eager_gpu", [(4, 4, False, False), (4, 4, False, True), (3, 3, True, False), (3, 3, True, True), (1, 7, False, False)])
def test_seal_is_the_quantizer(gpu, dtype, rbits, tbits, packed, eager_gpu):
    c = Cache(gpu, [1, 128, 300, 700, 0], [0, 0, 0, 0, 0], [0, 0, 1, 2, 0], 2, 2, dtype, rbits, tbits, packed)
    before = [t.clone() for t in (c.pool.codes, *c.pool.meta)]
    seal_pages(c.pool, c.batch, eager_gpu=eager_gpu)
    for b, n in enumerate(c.kv):
        new = slice(c.sealed[b], n // PAGE)
        if new.stop > new.start:
            want = quantize_and_pack_nbit(c.raw[b][None, :, new.start * PAGE:new.stop * PAGE].contiguous(), rbits, tbits, packed=packed, eager_gpu=eager_gpu)
            to = c.pages[b, new].long()
            for t, old, w in zip((c.pool.codes, *c.pool.meta), before, want):
                assert torch.equal(t[to], w[0].transpose(0, 1))
                old[to] = t[to]
    for t, old in zip((c.pool.codes, *c.pool.meta), before):                # and nothing else
        assert torch.equal(t.nan_to_num(3.0) if t.is_floating_point() else t, old.nan_to_num(3.0) if t.is_floating_point() else old)


def test_seal_without_a_page(gpu):
    c = Cache(gpu, [300], [0], [0], 2, 2, torch.float16)
    before = c.pool.codes.clone()
    open_pages, pages = c.open_pages.clone(), c.pages.clone()
    open_pages[0, 0], pages[0, 1] = -1, 99
    seal_pages(c.pool, c.batch_of(pages, open_pages))
    assert torch.equal(c.pool.codes, before)


# ---------------------------------------------------------------- eviction
@pytest.mark.parametrize("B,Nk,W,keep,sinks", [(1, 1, 1, 1, 0), (5, 2, 7, 3, 1), (9, 8, 40, 40, 2), (7, 3, 64, 17, 4), (4, 2, 1025, 500, 1), (3, 1, 2500, 1, 1), (2, 4, 16384, 9000, 3)])
def test_evict(gpu, B, Nk, W, keep, sinks):
    """Ties (few different weights), zeros of either sign, infinities, sequences of no page and of fewer than stay, holes among the open pages."""
    r = random.Random(W)
    n = [W] + [r.randint(0, W) for _ in range(B - 1)]
    for levels in (3, 1 << 20):
        weights = torch.tensor([r.choice([-0.0, 0.0, 1e-30, float("inf")]) if r.random() < 0.1 else r.randrange(levels) / 7 for _ in range(B * Nk * W)],
                               dtype=torch.float32).view(B, Nk, W)
        pages = torch.tensor([[r.randrange(1 << 20) if j < n[b] or r.random() < 0.5 else -1 for j in range(W)] for b in range(B)], dtype=torch.int32)
        kv = [PAGE * x + r.randrange(PAGE) for x in n]
        kv_max = PAGE * W
        batch = PageBatch(None, torch.tensor([min(x, kv_max) for x in kv], dtype=torch.int32, device=gpu), torch.tensor(n, dtype=torch.int32, device=gpu), pages.to(gpu), None, 1, kv_max)
        got, left, freed = evict_pages(weights.to(gpu), batch, keep, sinks)
        want = evicted(weights.tolist(), pages.tolist(), n, [min(x, kv_max) for x in kv], keep, sinks)
        assert got.pages.tolist() == want[0] and got.n_sealed.tolist() == want[1] and got.kv_len.tolist() == want[2]
        assert torch.equal(left.cpu(), torch.tensor(want[3], dtype=torch.float32)) and freed.tolist() == want[4]


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_server_step_by_step(gpu, dtype):
    """Two sequences in portions and tokens over one pool: rows appended, attended to, pages sealed as they fill, and once the least attended pages evicted;
    against the sequences' tokens kept beside."""
    N, Nk, rep, pool = 8, 2, 4, PagePool.empty(24, 12, 2, dtype, gpu)
    g = torch.Generator(device=gpu).manual_seed(3)
    f = 1e4 ** (-torch.arange(64, device=gpu) / 64)
    angle = torch.arange(2000, device=gpu)[:, None] * f
    cos, sin = (torch.cat([t, t], -1).to(dtype) for t in (angle.cos(), angle.sin()))
    free, free_open = list(range(24)), list(range(12))
    pages, opened, kv, sealed, seen = [[], []], [[], []], [0, 0], [0, 0], [0, 0]
    keys, values = [torch.empty(Nk, 0, 128, dtype=F64, device=gpu)] * 2, [torch.empty(Nk, 0, 128, dtype=F64, device=gpu)] * 2
    weights = torch.zeros(2, Nk, 16, device=gpu)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=gpu)

    def table(rows, W):
        return ints([r + [-1] * (W - len(r)) for r in rows])
    for step, new in enumerate([[200, 0], [130, 300], [1, 1], [1, 90], [60, 1], [1, 1]]):
        for b in range(2):
            kv[b] += new[b]
            while len(pages[b]) * PAGE < kv[b]:
                pages[b].append(free.pop(7 % len(free)))
            while (sealed[b] + len(opened[b])) * PAGE < kv[b]:
                opened[b].append(free_open.pop(3 % len(free_open)))
        T = sum(new)
        batch = PageBatch(ints([0, new[0], T]), ints(kv), ints(sealed), table(pages, 16), table(opened, 8), max(new), max(kv))
        qkv = torch.randn(T, 12 * 128, generator=g, device=gpu).to(dtype)
        positions = ints([seen[b] + t for b in range(2) for t in range(new[b])])
        w = torch.ones(128, device=gpu, dtype=dtype)
        q = qk_norm_rope_append(qkv[:, :1024], qkv[:, 1024:1280], qkv[:, 1280:], cos, sin, pool, batch, q_norm=w, k_norm=w, positions=positions)
        out, lse = paged_attention(q, pool, batch, return_lse=True)
        weights = page_weights(q, lse, pool, batch, onto=weights)
        # the same beside: rows as they were written
        for b in range(2):
            seen[b] += new[b]
            rows = []
            for j in range(kv[b] - new[b], kv[b]):
                rows.append((pool.keys[opened[b][j // PAGE - sealed[b]], :, j % PAGE], pool.values[pages[b][j // PAGE], :, j % PAGE]))
            if rows:
                keys[b] = torch.cat([keys[b], torch.stack([r[0] for r in rows], 1).to(F64)], 1)
                values[b] = torch.cat([values[b], torch.stack([r[1] for r in rows], 1).to(F64)], 1)
        c = Cache.__new__(Cache)
        c.kv, c.new, c.sealed, c.N, c.Nk, c.dtype, c.gpu, c.keys, c.values, c.q_start, c.q, c.T, c.mask = (kv, new, sealed, N, Nk, dtype, gpu, keys, values, batch.q_start,
                                                                                                         q, T, None)
        want, bound, want_lse, lse_bound = c.attention()
        near(out, want, bound)
        near(lse, want_lse, lse_bound)
        seal_pages(pool, batch)
        for b in range(2):
            for j in range(sealed[b], kv[b] // PAGE):
                p = pages[b][j]
                part = [pool.codes[p][:, None]] + [m[p][:, None] for m in pool.meta]
                keys[b][:, j * PAGE:(j + 1) * PAGE] = dequantized([t[None] for t in part], 4, 4)[0]
                free_open.append(opened[b].pop(0))
            sealed[b] = kv[b] // PAGE
        if step == 3:
            batch = PageBatch(None, ints(kv), ints(sealed), table(pages, 16), None, 1, PAGE * 16)
            left = weights.double().sum(1).float().tolist()
            closed, weights, freed = evict_pages(weights, batch, keep=2)
            for b in range(2):
                stay = sorted([0] + sorted(range(1, sealed[b]), key=lambda j: (-left[b][j], j))[:1]) if sealed[b] > 2 else list(range(sealed[b]))
                gone = [p for p in freed[b].tolist() if p >= 0]
                assert gone == [pages[b][j] for j in range(sealed[b]) if j not in stay]
                tokens = torch.tensor([j * PAGE + i for j in stay for i in range(PAGE)] + list(range(sealed[b] * PAGE, kv[b])), device=gpu)
                keys[b], values[b] = keys[b][:, tokens], values[b][:, tokens]
                pages[b] = [p for p in closed.pages[b].tolist() if p >= 0]
                free += gone
                kv[b], sealed[b] = int(closed.kv_len[b]), int(closed.n_sealed[b])
    assert seen == [393, 393] and min(kv) < 393


def test_a_captured_step_is_replayed_over_other_tables(gpu):
    """Rows and attention in a graph: counts, tables and rows change between the replays, with eager work among them."""
    dtype, N, Nk = torch.bfloat16, 8, 2
    cases = [Cache(gpu, kv, [1, 1], s, N, Nk, dtype, seed=i, wide=8 - max(-(-n // PAGE) for n in kv))
             for i, (kv, s) in enumerate([([300, 900], [2, 7]), ([1, 640], [0, 4]), ([1000, 129], [6, 1])])]
    pool = cases[0].pool
    size = [max(getattr(c.pool, n).shape[0] for c in cases) for n in ("keys", "values")]
    pool = PagePool.empty(size[1], size[0], Nk, dtype, gpu)
    width = max(c.open_pages.shape[1] for c in cases)
    q_start, kv_len, n_sealed = (torch.zeros(n, dtype=torch.int32, device=gpu) for n in (3, 2, 2))
    pages, open_pages = torch.full((2, 8), -1, dtype=torch.int32, device=gpu), torch.full((2, width), -1, dtype=torch.int32, device=gpu)
    batch = PageBatch(q_start, kv_len, n_sealed, pages, open_pages, 1, 1024)
    rows = torch.zeros(2, 12 * 128, dtype=dtype, device=gpu)
    cos, sin = torch.ones(1024, 128, device=gpu, dtype=dtype), torch.zeros(1024, 128, device=gpu, dtype=dtype)

    def load(c):
        for n in ("keys", "values", "codes"):
            getattr(pool, n)[:getattr(c.pool, n).shape[0]] = getattr(c.pool, n)
        for to, m in zip(pool.meta, c.pool.meta):
            to[:m.shape[0]] = m
        q_start.copy_(c.q_start), kv_len.copy_(c.batch.kv_len), n_sealed.copy_(c.batch.n_sealed), pages.copy_(c.pages)
        open_pages.fill_(-1)
        open_pages[:, :c.open_pages.shape[1]] = c.open_pages
        rows.copy_(torch.randn(2, 12 * 128, generator=torch.Generator(device=gpu).manual_seed(c.kv[0]), device=gpu))

    def step():
        q = qk_norm_rope_append(rows[:, :1024], rows[:, 1024:1280], rows[:, 1280:], cos, sin, pool, batch)
        return paged_attention(q, pool, batch)
    load(cases[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for c in cases + cases[:1]:
        load(c)
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step())
        for b in range(2):
            c.keys[b][:, -1] = rows[b, 1024:1280].view(Nk, 128).to(F64)
            c.values[b][:, -1] = rows[b, 1280:].view(Nk, 128).to(F64)
        c.q = rows[:, :1024].reshape(2, N, 128)
        want, bound, _, _ = c.attention()
        near(got, want, bound)


def test_on_another_stream(gpu):
    c = Cache(gpu, [2000, 300], [1, 1], [15, 2], 8, 2, torch.float16)
    here = paged_attention(c.q, c.pool, c.batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = paged_attention(c.q, c.pool, c.batch)
    torch.cuda.synchronize()
    assert torch.equal(here, there)
