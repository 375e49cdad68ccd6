"""Append into a paged cache (rotation on the way) and the one-token attention over it, against
plain implementations in 64 bits.

Tolerances (u = eps / 2 of the dtype, the worst case of one rounding; the kernels work in fp32):
* a rotated element x c - y s: two products and a difference, 3 roundings of at most
  2^-24 (|x| + |y|), then one rounding to the dtype: u |ref| + 2^-22 (|x| + |y|), plus half the
  smallest fp16 step, 2^-25.
* the attention: a score sums D products in fp32, off by at most D 2^-23 sum |q k| scale =: ds
  (2^-23: matrix instructions may round their sums toward zero), so a weight exp(s - max) is off
  by at most 2 ds + 2^-20 of itself, is held in two 16-bit parts (2^-16), and n of them are added
  (n 2^-24). Normalised weights sum to 1, so the output is off by at most
  2 (2 ds + 2^-20 + 2^-16 + n 2^-24) max |v|, then u |ref| for the rounding.
"""
import math

import pytest
import torch

from analysis_spec_b200 import _ops
from analysis_spec_b200.paged_cache import PagedKVCache, paged_append, paged_attention, rotation_tables
from analysis_spec_b200.token_logprobs import token_logprobs

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def randn(*shape, dtype, g):
    return torch.randn(*shape, device='cuda', generator=g).to(dtype)


def pools(pages, hkv, page, dim, dtype, g, fill=math.nan):
    return (torch.full((pages, hkv, page, dim), fill, device='cuda', dtype=dtype),
            torch.full((pages, hkv, page, dim), fill, device='cuda', dtype=dtype))


def turned(x, cos, sin, interleaved):
    """x (..., dim) float64, cos / sin (..., rot / 2); returns (rotated, |x| + |y| of each element)."""
    half = cos.shape[-1]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out, size = x.clone(), x.abs()
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return out, size


def check_rounded(got, ref, size, dtype):
    u = torch.finfo(dtype).eps / 2
    tol = u * ref.abs() + 2.0 ** -22 * size + (2.0 ** -25 if dtype == torch.float16 else 0)
    bad = ((got.double() - ref).abs() > tol)
    assert not bad.any(), (bad.sum().item(), (got.double() - ref).abs().max().item())


# ---- append ------------------------------------------------------------------------------------

def run_append(batch, rows, hq, hkv, dim, rot, page, past, dtype, interleaved, ragged, placed, query=True, seed=0):
    g = gen(seed)
    per = -(-(past + rows) // page)
    total = batch * per + 2
    kp, vp = pools(total, hkv, page, dim, dtype, g)
    table = torch.randperm(total, device='cuda', generator=g)[:batch * per].view(batch, per).contiguous()
    # one fused projection output, sliced and viewed by head: strided, not dense
    fused = randn(batch, rows, (hq + 2 * hkv) * dim, dtype=dtype, g=g)
    q, k, v = (x.unflatten(-1, (-1, dim)).transpose(1, 2) for x in fused.split((hq * dim, hkv * dim, hkv * dim), -1))
    starts = torch.randint(0, past + 1, (batch,), device='cuda', generator=g)
    counts = torch.randint(0, rows + 1, (batch,), device='cuda', generator=g) if ragged else None
    positions = torch.randint(0, 50, (batch, rows), device='cuda', generator=g) if placed else None
    tables = rotation_tables(max(past + rows, 50), rot, theta=5000.0) if rot else None
    out = paged_append(k, v, kp, vp, table, starts, counts=counts, query=q if query else None, rotation=tables,
                       positions=positions, interleaved=interleaved)
    assert _ops.device_error() is None
    want_k, want_v = (torch.full(kp.shape, math.nan, device='cuda', dtype=torch.float64) for _ in range(2))
    size_k = torch.zeros_like(want_k)
    for b in range(batch):
        n = rows if counts is None else int(counts[b])
        slot = int(starts[b]) + torch.arange(n, device='cuda')
        where = slot if positions is None else positions[b, :n]
        kk, qq = k[b, :, :n].double(), q[b, :, :n].double()
        ks, qs = kk.abs(), qq.abs()
        if rot:
            c, s = tables[0][where].double(), tables[1][where].double()
            (kk, ks), (qq, qs) = turned(kk, c, s, interleaved), turned(qq, c, s, interleaved)
        at = table[b][slot // page]
        want_k[at, :, slot % page] = kk.transpose(0, 1)
        size_k[at, :, slot % page] = ks.transpose(0, 1)
        want_v[at, :, slot % page] = v[b, :, :n].double().transpose(0, 1)
        if query:
            check_rounded(out[b, :, :n], qq, qs, dtype)
            assert not out[b, :, n:].any()  # padding rows: zeros
    assert torch.equal(vp.double().nan_to_num(9e9), want_v.nan_to_num(9e9))  # copied; nothing else touched
    assert torch.equal(kp.isnan(), want_k.isnan())
    check_rounded(kp.double().nan_to_num(0.0), want_k.nan_to_num(0.0), size_k, dtype)
    if not query:
        assert out is None


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('batch,rows,hq,hkv,dim,rot,page,past', [
    (1, 1, 16, 2, 128, 128, 16, 0), (8, 1, 28, 4, 128, 128, 64, 700), (3, 61, 16, 2, 128, 128, 16, 100),
    (2, 37, 8, 8, 64, 32, 32, 5), (2, 5, 6, 3, 256, 256, 128, 300), (4, 7, 12, 1, 128, 64, 16, 40),
    (3, 4, 6, 2, 40, 20, 3, 11), (2, 9, 3, 1, 24, 14, 1, 6), (5, 1, 4, 4, 80, 80, 24, 60), (1, 300, 40, 8, 96, 96, 7, 9)])
def test_append_and_rotation(batch, rows, hq, hkv, dim, rot, page, past, dtype):
    run_append(batch, rows, hq, hkv, dim, rot, page, past, dtype, interleaved=False, ragged=rows > 1, placed=False)
    run_append(batch, rows, hq, hkv, dim, rot, page, past, dtype, interleaved=True, ragged=rows > 1, placed=True, seed=1)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('batch,rows,hq,hkv,dim,rot,page,past', [
    (40, 61, 16, 2, 128, 128, 16, 100), (3, 901, 4, 1, 64, 32, 8, 7), (2, 1300, 1, 1, 256, 256, 64, 0),
    (7, 400, 7, 3, 128, 96, 16, 20), (43, 61, 28, 4, 128, 128, 16, 9)])
def test_append_of_many_tokens(batch, rows, hq, hkv, dim, rot, page, past, dtype):
    """More tokens than the CTAs of 64 threads that run at once: a warp per token where heads are few."""
    run_append(batch, rows, hq, hkv, dim, rot, page, past, dtype, interleaved=False, ragged=True, placed=False)
    run_append(batch, rows, hq, hkv, dim, rot, page, past, dtype, interleaved=True, ragged=False, placed=True, seed=1,
               query=batch != 3)


def test_append_of_many_tokens_reports_bad_pages():
    """Sequence 1's second page is none of the pools', sequence 2 starts past the table: their tokens
    there are padding, every other one is stored."""
    g = gen(11)
    k, v = (randn(3, 2, 900, 128, dtype=torch.bfloat16, g=g) for _ in range(2))
    q = randn(3, 8, 900, 128, dtype=torch.bfloat16, g=g)
    kp, vp = pools(30, 2, 100, 128, torch.bfloat16, g)
    table = torch.arange(27, device='cuda').view(3, 9).contiguous()
    table[1, 1] = 30
    starts = torch.tensor([0, 0, 500], device='cuda')
    out = paged_append(k, v, kp, vp, table, starts, query=q, rotation=rotation_tables(900, 128))
    kind, where = _ops.device_error()
    assert kind == 'page table' and (where == 30 or 900 <= where < 1400)
    live = torch.ones(3, 900, dtype=torch.bool, device='cuda')
    live[1, 100:200] = False
    live[2, 400:] = False
    assert out.transpose(1, 2)[live].any(-1).all() and not out.transpose(1, 2)[~live].any()
    want = torch.full_like(vp, math.nan)
    for b in range(3):
        slot = int(starts[b]) + torch.arange(900, device='cuda')[live[b]]
        want[table[b][slot // 100], :, slot % 100] = v[b].transpose(0, 1)[live[b]]
    assert torch.equal(vp.nan_to_num(9.0), want.nan_to_num(9.0)) and torch.equal(kp.isnan(), want.isnan())


def test_append_without_rotation_or_query():
    run_append(3, 20, 4, 2, 128, 0, 16, 30, torch.bfloat16, False, True, False, query=False)
    run_append(3, 20, 4, 2, 128, 0, 16, 30, torch.bfloat16, False, False, False)
    run_append(2, 6, 4, 2, 72, 0, 5, 9, torch.float16, False, True, False)
    run_append(2, 6, 4, 2, 128, 128, 16, 9, torch.float16, False, True, True, query=False)


def test_append_strided_pages_positions_and_query_in_place():
    g = gen(3)
    both = torch.full((9, 2, 2, 16, 128), math.nan, device='cuda', dtype=torch.bfloat16)  # K and V of a page together
    flat = torch.full((9, 16, 2, 128), math.nan, device='cuda', dtype=torch.bfloat16)      # position before head
    table = torch.tensor([[8, 0, 3], [1, 7, 5]], device='cuda')[:, :2]                     # a wider table's columns
    q, k, v = (randn(2, h, 5, 128, dtype=torch.bfloat16, g=g) for h in (4, 2, 2))
    starts = torch.tensor([13, 0], device='cuda')
    tables = rotation_tables(64, 128)
    positions = torch.randint(0, 64, (5, 2), device='cuda', generator=g).T
    ref = paged_append(k, v, both[:, 0], both[:, 1], table, starts, query=q, rotation=tables, positions=positions)
    plain = pools(9, 2, 16, 128, torch.bfloat16, g)
    want = paged_append(k, v, *plain, table, starts, query=q, rotation=tables, positions=positions.contiguous())
    assert torch.equal(ref, want)
    for i in range(2):
        assert torch.equal(both[:, i].nan_to_num(9.0), plain[i].nan_to_num(9.0))
    q2 = q.clone()
    got = paged_append(k, v, flat.transpose(1, 2), plain[1], table, starts, query=q2, rotation=tables,
                       positions=positions, query_out=q2)
    assert got is q2 and torch.equal(q2, want)
    assert torch.equal(flat.transpose(1, 2).nan_to_num(9.0), plain[0].nan_to_num(9.0))
    assert _ops.device_error() is None


@pytest.mark.parametrize('dim', [128, 40])
def test_append_reports_what_it_cannot_place(dim):
    g = gen(4)
    k, v, q = (randn(3, 2, 4, dim, dtype=torch.bfloat16, g=g) for _ in range(3))
    tables = rotation_tables(30, dim)
    good = torch.tensor([[0], [1], [2]], device='cuda')

    def run(table, starts, positions=None):
        kp, vp = pools(3, 2, 16, dim, torch.bfloat16, g)
        out = paged_append(k, v, kp, vp, table, torch.tensor(starts, device='cuda'), query=q, rotation=tables,
                           positions=positions)
        return kp, vp, out, _ops.device_error()

    for bad in (3, -1, 1 << 40):  # a page outside the pools
        table = good.clone()
        table[1] = bad
        kp, vp, out, err = run(table, [0, 0, 0])
        assert err is not None and err[0] == 'page table'
        assert kp[1].isnan().all() and vp[1].isnan().all() and not out[1].any()
        assert not kp[0, :, :4].isnan().any() and out[2].any()
    kp, vp, out, err = run(good, [0, 14, -2])  # rows past the table's positions, and before the first
    assert err[0] == 'page table'
    assert not kp[1, :, 14:].isnan().any() and kp[1, :, :14].isnan().all() and not out[1, :, 2:].any()
    assert not kp[2, :, :2].isnan().any() and kp[2, :, 2:].isnan().all() and not out[2, :, :2].any()
    positions = torch.zeros(3, 4, dtype=torch.long, device='cuda')
    positions[0, 1], positions[2, 3] = 30, -1  # outside the rotation tables
    kp, vp, out, err = run(good, [0, 0, 0], positions)
    assert err[0] == 'rotation index'
    assert kp[0, :, 1].isnan().all() and vp[2, :, 3].isnan().all() and not out[0, :, 1].any()
    assert not kp[0, :, 2].isnan().any()
    assert _ops.device_error() is None


# ---- attention -----------------------------------------------------------------------------------

def filled(batch, hkv, dim, page, lengths, dtype, g, scale=1.0, extra=2, slack=0):
    """Pools that hold NaN wherever no live position is, and the table (entries past the length: -7)."""
    per = max(1, max(-(-n // page) for n in lengths)) + slack
    total = batch * (per - slack) + extra
    kp, vp = pools(total, hkv, page, dim, dtype, g)
    order = torch.randperm(total, device='cuda', generator=g)
    table = torch.full((batch, per), -7, dtype=torch.long, device='cuda')
    at = 0
    for b, n in enumerate(lengths):
        used = -(-n // page)
        table[b, :used] = order[at:at + used]
        at += used
        slot = torch.arange(n, device='cuda')
        where = table[b][slot // page]
        kp[where, :, slot % page] = scale * randn(n, hkv, dim, dtype=dtype, g=g)
        vp[where, :, slot % page] = randn(n, hkv, dim, dtype=dtype, g=g)
    return kp, vp, table


def check_attention(out, q, kp, vp, table, lengths, scale, page, dtype):
    batch, hq, _, dim = q.shape
    hkv = kp.shape[1]
    u = torch.finfo(dtype).eps / 2
    assert out.shape == (batch, 1, hq, dim)
    for b, n in enumerate(lengths):
        if n <= 0:
            assert not out[b].any()
            continue
        slot = torch.arange(n, device='cuda')
        where = table[b][slot // page]
        k = kp[where, :, slot % page].double().transpose(0, 1)
        v = vp[where, :, slot % page].double().transpose(0, 1)
        qq = q[b, :, 0].double().view(hkv, hq // hkv, dim)
        s = torch.einsum('hgd,hnd->hgn', qq, k) * scale
        ref = torch.einsum('hgn,hnd->hgd', torch.softmax(s, -1), v)
        ds = dim * 2.0 ** -23 * torch.einsum('hgd,hnd->hgn', qq.abs(), k.abs()).amax(-1, keepdim=True) * abs(scale)
        vmax = v.abs().amax(1, keepdim=True)
        tol = u * ref.abs() + 2 * (2 * ds + 2.0 ** -20 + 2.0 ** -16 + n * 2.0 ** -24) * vmax
        err = (out[b, 0].double().view_as(ref) - ref).abs()
        assert (err <= tol).all(), (b, n, (err - tol).max().item(), err.max().item())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('hq,hkv,dim,page,lengths', [
    (16, 2, 128, 16, [1, 0, 200, 15, 16, 17, 33, 640]), (28, 4, 128, 64, [1000, 63, 64, 65, 129]),
    (40, 8, 128, 128, [4097]), (8, 8, 64, 32, [5, 90, 0, 31, 32, 257]), (12, 1, 128, 16, [100, 1500]),
    (16, 1, 64, 16, [77, 300]), (4, 2, 256, 16, [1, 19, 500]), (20, 1, 128, 32, [40, 333]), (32, 1, 256, 64, [130]),
    (6, 2, 128, 1, [50, 3]), (5, 1, 64, 3, [1, 100, 7]), (7, 7, 128, 24, [230, 24, 25]), (14, 2, 128, 8, [64, 9]),
    (8, 1, 128, 32, list(range(1, 75, 2))), (4, 4, 64, 16, [700, 0, 90] * 5), (2, 2, 256, 8, [300] * 23),
    (6, 2, 40, 16, [19, 100]), (3, 1, 80, 5, [33, 0, 4]), (2, 2, 192, 16, [70]), (1, 1, 8, 2, [9])])
def test_attention_over_pages(hq, hkv, dim, page, lengths, dtype):
    batch = len(lengths)
    # a table as wide as the lengths (a cluster per item), and one of 13000 positions (equal shares)
    for slack in (0, -(-13000 // page)):
        g = gen(hq * 7 + page)
        kp, vp, table = filled(batch, hkv, dim, page, lengths, dtype, g, slack=slack)
        q = randn(batch, 1, hq * dim, dtype=dtype, g=g).view(batch, 1, hq, dim).transpose(1, 2)
        out = paged_attention(q, kp, vp, table, torch.tensor(lengths, device='cuda'))
        check_attention(out, q, kp, vp, table, lengths, dim ** -0.5, page, dtype)
        assert _ops.device_error() is None


@pytest.mark.parametrize('hq,hkv,batch', [(8, 1, 1), (16, 2, 3), (4, 4, 40), (28, 4, 70)])
def test_attention_splits_long_and_ragged_lengths(hq, hkv, batch):
    """One long sequence beside short ones: shares of it end anywhere inside a page or a tile."""
    g = gen(hq + batch)
    lengths = [int(x) for x in torch.randint(0, 400, (batch,), generator=torch.Generator().manual_seed(batch))]
    lengths[batch // 2] = 9001
    kp, vp, table = filled(batch, hkv, 128, 16, lengths, torch.bfloat16, g)
    q = randn(batch, hq, 1, 128, dtype=torch.bfloat16, g=g)
    n = torch.tensor(lengths, device='cuda')
    out = paged_attention(q, kp, vp, table, n)
    check_attention(out, q, kp, vp, table, lengths, 128 ** -0.5, 16, torch.bfloat16)
    assert all(torch.equal(out, paged_attention(q, kp, vp, table, n)) for _ in range(3))  # same order, same bits
    assert _ops.device_error() is None


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('scale', [8.0, -1.0, 0.0])
def test_attention_peaked_flat_and_negative_scales(dtype, scale):
    g = gen(5)
    lengths = [300, 47]
    kp, vp, table = filled(2, 2, 128, 16, lengths, dtype, g, scale=0.2)
    q = randn(2, 16, 1, 128, dtype=dtype, g=g)
    out = paged_attention(q, kp, vp, table, torch.tensor(lengths, device='cuda'), scale)
    check_attention(out, q, kp, vp, table, lengths, scale, 16, dtype)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [4, 8, 24, 56, 72, 80, 96, 112, 120, 136, 160, 192, 248])
def test_attention_head_dims_between(dim, dtype):
    """Head dims that the kernels read as the next one they are built for, with zeros behind; pools whose
    rows lie side by side, so that a row's end is the next one's beginning."""
    lengths = [1, 0, 130, 47, 700]
    for hq, hkv, page, slack in ((6, 2, 16, 0), (20, 2, 5, 0), (3, 3, 64, 400), (12, 1, 8, 2000)):
        g = gen(dim + hq)
        kp, vp, table = filled(5, hkv, dim, page, lengths, dtype, g, slack=slack)
        q = randn(5, 1, hq * dim, dtype=dtype, g=g).view(5, 1, hq, dim).transpose(1, 2)
        out = torch.full((6, 1, hq, dim), 7.0, dtype=dtype, device='cuda')
        paged_attention(q, kp, vp, table, torch.tensor(lengths, device='cuda'), out=out[:5])
        check_attention(out[:5], q, kp, vp, table, lengths, dim ** -0.5, page, dtype)
        assert (out[5] == 7.0).all() and _ops.device_error() is None


def test_attention_infinite_keys_of_a_dim_between():
    """fp32 keys of -inf are summed term by term: over the row's own dims only."""
    g = gen(12)
    kp, vp, table = filled(1, 2, 80, 16, [90], torch.float32, g)
    q = randn(1, 4, 1, 80, dtype=torch.float32, g=g).abs()
    kp[table[0, 1], :, 3] = -math.inf
    out = paged_attention(q, kp, vp, table, torch.tensor([90], device='cuda'))
    keep = torch.arange(90, device='cuda') != 19
    where, row = table[0][torch.arange(90, device='cuda')[keep] // 16], torch.arange(90, device='cuda')[keep] % 16
    kp2, vp2 = (torch.zeros(6, 2, 16, 80, device='cuda') for _ in range(2))
    slot = torch.arange(89, device='cuda')
    kp2[slot // 16, :, slot % 16], vp2[slot // 16, :, slot % 16] = kp[where, :, row], vp[where, :, row]
    check_attention(out, q, kp2, vp2, torch.arange(6, device='cuda')[None], [89], 80 ** -0.5, 16, torch.float32)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n', [5000, 60000])
@pytest.mark.parametrize('dim', [64, 128])
def test_attention_sums_many_small_weights(dtype, n, dim):
    """One key takes nearly all the weight and n - 1 have e^-18 of it each (2^-26, below fp16's smallest
    step): only they have values. Scores are exact but for the factor scale log2(e), off by 2^-23 of
    |s| = 26; the weights are summed in fp32 (n 2^-23 of the sum at most) and fp16 drops 2^-36 of the
    largest weight of each."""
    k = torch.zeros(n, dim, dtype=dtype, device='cuda')
    k[1:, 0] = -18.0
    v = torch.ones(n, dim, dtype=dtype, device='cuda')
    v[0] = 0
    pages = -(-n // 16)
    kp, vp = torch.zeros(2, pages, 1, 16, dim, dtype=dtype, device='cuda')
    kp.view(-1, dim)[:n], vp.view(-1, dim)[:n] = k, v
    q = torch.zeros(1, 5, 1, dim, dtype=dtype, device='cuda')
    q[..., 0] = 1
    table = torch.arange(pages, device='cuda')[None]
    out = paged_attention(q, kp, vp, table, torch.tensor([n], device='cuda'), 1.0).double()
    mass = (n - 1) * math.exp(-18)
    ref = mass / (1 + mass)
    u = torch.finfo(dtype).eps / 2
    assert ((out - ref).abs() <= ref * (u + 2.0 ** -16 + 26 * 2.0 ** -22 + n * 2.0 ** -23) + n * 2.0 ** -36).all(), (
        out[0, 0, 0, 0].item(), ref)


def test_attention_rising_scores_and_lowest_values():
    """Every key beats the ones before it (the running maximum moves each step); keys whose score is
    hugely negative; a key that holds -inf products (weight 0); one with NaN (its row is NaN)."""
    g = gen(6)
    n, dim = 1111, 128
    kp, vp, table = filled(1, 1, dim, 16, [n], torch.float32, g)
    q = torch.zeros(1, 2, 1, dim, device='cuda')
    q[0, 0, 0, 0], q[0, 1, 0, 1] = 1.0, 1.0
    slot = torch.arange(n, device='cuda')
    kp[table[0][slot // 16], 0, slot % 16, 0] = slot.float()
    low = torch.full((n,), -1e30, device='cuda')
    low[700] = 0.5
    kp[table[0][slot // 16], 0, slot % 16, 1] = low
    out = paged_attention(q, kp, vp, table, torch.tensor([n], device='cuda'), 1.0)
    v = vp[table[0][slot // 16], 0, slot % 16].double()
    ref = torch.softmax(slot.double(), 0) @ v
    assert (out[0, 0, 0].double() - ref).abs().max() < 1e-4 * v.abs().max()  # scores to 1111: 2^-14 of them, once
    # one key has all the weight, exactly 1; its value enters as two tf32 parts, the second cut to 11 of
    # its at most 13 bits: 2^-11 2^-11 = 2^-22 of the value is left out at most
    assert ((out[0, 0, 1].double() - v[700]).abs() <= 2.0 ** -22 * v[700].abs()).all()
    kp[table[0][0], 0, 3, 1] = -math.inf
    out = paged_attention(q[:, 1:], kp, vp, table, torch.tensor([n], device='cuda'), 1.0)[0, 0, 0]
    assert ((out.double() - v[700]).abs() <= 2.0 ** -22 * v[700].abs()).all()
    kp[table[0][0], 0, 3, 1] = math.nan
    assert paged_attention(q[:, 1:], kp, vp, table, torch.tensor([n], device='cuda'), 1.0).isnan().all()
    # keys of -inf alone leave nothing to attend: zeros, as a length of 0
    kp[:, :, :, 1] = -math.inf
    assert not paged_attention(q[:, 1:], kp, vp, table, torch.tensor([40], device='cuda'), 1.0).any()


@pytest.mark.parametrize('dim,dtype', [(128, torch.bfloat16), (64, torch.float32), (40, torch.float16)])
def test_attention_strided_pages_and_query(dim, dtype):
    g = gen(7)
    lengths = [70, 33, 128]
    kp, vp, table = filled(3, 2, dim, 16, lengths, dtype, g)
    both = torch.stack((kp, vp), 1)                                 # K and V of a page together
    flat_k, flat_v = (p.transpose(1, 2).contiguous().transpose(1, 2) for p in (kp, vp))  # position before head
    fused = randn(3, 1, 10 * dim, dtype=dtype, g=g)
    q = fused[..., :8 * dim].view(3, 1, 8, dim).transpose(1, 2)     # queries of a fused projection
    n = torch.tensor(lengths, device='cuda')
    wide = torch.cat((table, table), 1)[:, :table.shape[1]]
    ref = paged_attention(q.contiguous(), kp, vp, table, n)
    check_attention(ref, q, kp, vp, table, lengths, dim ** -0.5, 16, dtype)
    assert torch.equal(paged_attention(q, both[:, 0], both[:, 1], wide, n), ref)
    assert torch.equal(paged_attention(q, flat_k, flat_v, table, n), ref)
    odd = torch.zeros(both.numel() + 1, device='cuda', dtype=dtype)[1:].view(both.shape)  # off 16-byte alignment
    odd.copy_(both)
    check_attention(paged_attention(q, odd[:, 0], odd[:, 1], table, n), q, kp, vp, table, lengths, dim ** -0.5, 16, dtype)
    out = torch.full((3, 1, 8, dim), 7.0, device='cuda', dtype=dtype)
    assert paged_attention(q, kp, vp, table, n, out=out) is out and torch.equal(out, ref)


@pytest.mark.parametrize('dim', [128, 40])
def test_attention_reports_bad_pages_and_lengths(dim):
    g = gen(8)
    kp, vp, table = filled(3, 2, dim, 16, [64, 64, 64], torch.bfloat16, g)
    q = randn(3, 4, 1, dim, dtype=torch.bfloat16, g=g)
    n = torch.tensor([64, 64, 64], device='cuda')
    ref = paged_attention(q, kp, vp, table, n)
    assert _ops.device_error() is None
    for bad in (-1, kp.shape[0], 1 << 45):
        t = table.clone()
        t[1, 2] = bad
        out = paged_attention(q, kp, vp, t, n)
        err = _ops.device_error()
        assert err is not None and err[0] == 'page table'
        assert torch.equal(out[0], ref[0]) and torch.equal(out[2], ref[2])
        # the positions of that page are not attended
        keep = torch.cat((table[1:2, :2], table[1:2, 3:]), 1)
        want = paged_attention(q[1:2], kp, vp, keep, torch.tensor([48], device='cuda'))
        assert (out[1] - want[0]).abs().max() <= 2.0 ** -7 * want.abs().max()  # other order of sums: 2 roundings
    out = paged_attention(q, kp, vp, table, torch.tensor([65, 64, -3], device='cuda'))  # past the table; below zero
    assert _ops.device_error()[0] == 'page table'
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1]) and not out[2].any()


def test_pools_beyond_32_bit_offsets():
    """Pools of more than 2^31 elements, addressed at their far end."""
    page, dim = 16, 128
    pages = (2 ** 31 // (page * dim)) + 40
    kp = torch.empty(pages, 1, page, dim, device='cuda', dtype=torch.bfloat16)
    vp = torch.empty_like(kp)
    g = gen(9)
    table = torch.tensor([[pages - 1, 5, pages - 30]], device='cuda')
    k, v = (randn(1, 1, 45, dim, dtype=torch.bfloat16, g=g) for _ in range(2))
    q = randn(1, 8, 1, dim, dtype=torch.bfloat16, g=g)
    paged_append(k, v, kp, vp, table, torch.zeros(1, dtype=torch.long, device='cuda'))
    assert torch.equal(kp[pages - 1, 0], k[0, 0, :16]) and torch.equal(vp[pages - 30, 0, :13], v[0, 0, 32:])
    out = paged_attention(q, kp, vp, table, torch.tensor([45], device='cuda'))
    small = paged_attention(q, kp[-40:], vp[-40:], table * 0 + torch.tensor([[39, 0, 10]], device='cuda'),
                            torch.tensor([16], device='cuda'))
    check_attention(small, q, kp[-40:], vp[-40:], torch.tensor([[39]], device='cuda'), [16], dim ** -0.5, page,
                    torch.bfloat16)
    check_attention(out, q, kp, vp, table, [45], dim ** -0.5, page, torch.bfloat16)
    assert _ops.device_error() is None


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('slack', [0, 800])
def test_streams_and_graphs(dtype, slack):
    """A side stream, and two captured graphs of the same buffers replayed on two streams at once,
    with a cluster per item and with equal shares and their join."""
    g = gen(10)
    lengths = [3000, 17, 900]
    kp, vp, table = filled(3, 2, 128, 16, lengths, dtype, g, slack=slack)
    n = torch.tensor(lengths, device='cuda')
    qs = [randn(3, 16, 1, 128, dtype=dtype, g=g) for _ in range(2)]
    want = [paged_attention(q, kp, vp, table, n) for q in qs]
    check_attention(want[0], qs[0], kp, vp, table, lengths, 128 ** -0.5, 16, dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(paged_attention(qs[0], kp, vp, table, n), want[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(q, kp, vp, table, n))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(10):
                    graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    n.copy_(torch.tensor([5, 1, 0]))  # lengths are read on the device at each replay
    graphs[0].replay()
    torch.cuda.synchronize()
    check_attention(outs[0], qs[0], kp, vp, table, [5, 1, 0], 128 ** -0.5, 16, dtype)


def test_empty_calls():
    kp, vp = pools(1, 2, 16, 128, torch.bfloat16, None)
    table = torch.zeros(0, 1, dtype=torch.long, device='cuda')
    none = torch.zeros(0, dtype=torch.long, device='cuda')
    assert paged_attention(kp.new_zeros(0, 4, 1, 128), kp, vp, table, none).shape == (0, 1, 4, 128)
    k = kp.new_zeros(0, 2, 3, 128)
    assert paged_append(k, k, kp, vp, table, none) is None
    k = kp.new_zeros(2, 2, 0, 128)
    two = torch.zeros(2, dtype=torch.long, device='cuda')
    assert paged_append(k, k, kp, vp, two[:, None], two, query=k).shape == k.shape
    assert kp.isnan().all()


# ---- together --------------------------------------------------------------------------------------

def test_decode_loop_with_release_and_admission():
    """Prompts of unequal length, decode steps, a release and an admission, and the greedy token's
    log-probability of each step, against dense 64-bit attention over each sequence's own rows."""
    g = gen(11)
    hq, hkv, dim, page, vocab = 8, 2, 128, 16, 500
    dtype, scale = torch.bfloat16, 128 ** -0.5
    cache = PagedKVCache(40, page, batch_capacity=4, max_length=160)
    tables = rotation_tables(160, dim)
    head = randn(hq * dim, vocab, dtype=dtype, g=g) * 0.1
    history = []  # per live sequence: [(k rotated, v)] per layer

    def forward(counts, first, rows):
        batch = len(counts)
        cache.begin(counts, first)
        for layer in range(2):
            q, k, v = (randn(batch, h, rows, dim, dtype=dtype, g=g) for h in (hq, hkv, hkv))
            starts = [cache.lengths[first + b] - counts[b] for b in range(batch)]
            qr = cache.append(k, v, layer, query=q, rotation=tables)
            kp, vp = cache._pools[layer]
            for b in range(batch):
                seq = history[first + b][layer]
                at = cache.page_table()[first + b]
                slot = starts[b] + torch.arange(counts[b], device='cuda')
                kk, size = turned(k[b, :, :counts[b]].double(), tables[0][slot].double(), tables[1][slot].double(), False)
                check_rounded(kp[at[slot // page], :, slot % page].transpose(0, 1), kk, size, dtype)
                seq.append((kp[at[slot // page], :, slot % page], v[b, :, :counts[b]].transpose(0, 1)))
            if rows == 1:
                out = cache.attend(qr, layer, scale)
                for b in range(batch):
                    kk = torch.cat([x[0] for x in history[first + b][layer]])
                    vv = torch.cat([x[1] for x in history[first + b][layer]])
                    n = kk.shape[0]
                    assert n == cache.lengths[first + b]
                    # the cache holds this sequence's own rows: a one-page pool of them
                    check_attention(out[b:b + 1], qr[b:b + 1], kk.transpose(0, 1)[None], vv.transpose(0, 1)[None],
                                    torch.zeros(1, 1, dtype=torch.long, device='cuda'), [n], scale, n, dtype)
        if rows == 1:
            logits = (out.reshape(batch, -1) @ head).float()
            top = token_logprobs(logits, top=1)
            again = token_logprobs(logits, top.top_ids[:, 0])
            assert torch.equal(top.top_ids[:, 0], logits.argmax(-1))
            assert torch.equal(again.logprobs, top.top_logprobs[:, 0])
            ref = torch.log_softmax(logits.double(), -1).amax(-1)
            spread = (logits.amax() - logits.amin()).item()
            assert (again.logprobs.double() - ref).abs().max() <= 2.0 ** -21 * (1 + spread) + (vocab + 32) * 2.0 ** -24

    def admit(lengths):
        first = cache.admit(len(lengths))
        history.extend([[[], []] for _ in lengths])
        forward(lengths, first, max(lengths))

    admit([17, 1, 50])
    for _ in range(3):
        forward([1] * 3, 0, 1)
    keep = cache.release([False, True, False])
    assert keep == [0, 2]
    history[:] = [history[i] for i in keep]
    forward([1, 1], 0, 1)
    admit([33, 16])
    for _ in range(2):
        forward([1] * 4, 0, 1)
    assert cache.lengths == [23, 56, 35, 18] and cache.free_pages == 40 - (2 + 4 + 3 + 2)
    assert _ops.device_error() is None
    cache.reset()
    assert cache.free_pages == 40 and not cache.lengths


def test_transformers_model_decodes_through_pages():
    """A random-weight Qwen2: right-padded prompts and decode steps through PagedKVCache and the
    registered attention, against transformers' own cache and SDPA one sequence at a time."""
    from transformers import DynamicCache, Qwen2Config, Qwen2ForCausalLM
    from analysis_spec_b200.tree_attention import register
    name = register()
    torch.manual_seed(0)
    cfg = Qwen2Config(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=512, rms_norm_eps=1e-6,
                      tie_word_embeddings=False)
    cfg._attn_implementation = 'sdpa'
    model = Qwen2ForCausalLM(cfg).to('cuda', torch.bfloat16).eval()

    def use(impl):
        model.config._attn_implementation = impl
        for layer in model.model.layers:
            layer.self_attn.config._attn_implementation = impl

    prompts, steps = [7, 20, 13], 4
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 512, (3, 20), generator=g).cuda()
    new = torch.randint(0, 512, (3, steps), generator=g).cuda()
    want = []
    with torch.no_grad():
        for b, n in enumerate(prompts):
            past = DynamicCache()
            logits = [model(input_ids=ids[b:b + 1, :n], past_key_values=past, use_cache=True).logits[:, -1]]
            for t in range(steps):
                logits.append(model(input_ids=new[b:b + 1, t:t + 1], past_key_values=past, use_cache=True).logits[:, -1])
            want.append(torch.cat(logits).float())
        use(name)
        cache = PagedKVCache(16, 16, batch_capacity=3, max_length=64)
        cache.prompt_lengths(prompts)
        positions = torch.arange(20, device='cuda').expand(3, -1)
        out = model(input_ids=ids, position_ids=positions, past_key_values=cache, use_cache=True).logits.float()
        got = [[out[b, n - 1]] for b, n in enumerate(prompts)]
        for t in range(steps):
            before = torch.tensor(cache.lengths, device='cuda')[:, None]
            out = model(input_ids=new[:, t:t + 1], position_ids=before, past_key_values=cache, use_cache=True).logits
            for b in range(3):
                got[b].append(out[b, 0].float())
        assert cache.lengths == [n + steps for n in prompts]
        with pytest.raises(ValueError, match='one token'):
            model(input_ids=new[:, :2], position_ids=positions[:, :2], past_key_values=cache, use_cache=True)
    use('sdpa')
    for b in range(3):
        w, o = want[b], torch.stack(got[b])
        assert (o - w).abs().max() <= 0.06 * w.abs().max()  # two bf16 layers: some tens of roundings of 2^-8
    assert _ops.device_error() is None


@pytest.mark.parametrize('dtype', DTYPES)
def test_strides_of_single_entries_do_not_count(dtype):
    """A dimension of one entry may have any stride: the same kernels, the same bits."""
    g = gen(13)

    def odd(x, *dims):
        return x.as_strided(x.shape, [7 if d in dims else s for d, s in enumerate(x.stride())])

    for n, page in ((300, 16), (16, 16), (40, 1)):
        kp, vp, table = filled(1, 1, 128, page, [n], dtype, g, extra=0)
        dims = [1] + [0] * (kp.shape[0] == 1) + [2] * (page == 1)
        q = randn(1, 1, 1, 128, dtype=dtype, g=g)
        lengths = torch.tensor([n], device='cuda')
        want = paged_attention(q, kp, vp, table, lengths)
        assert torch.equal(paged_attention(odd(q, 0, 1, 2), odd(kp, *dims), odd(vp, *dims), table, lengths), want)
        new = [randn(1, 1, 1, 128, dtype=dtype, g=g) for _ in range(3)]
        starts = torch.tensor([n - 1], device='cuda')
        made = []
        for turn in (lambda x, *d: x, odd):
            k2, v2 = kp.clone(), vp.clone()
            out = paged_append(turn(new[0], 0, 1, 2), turn(new[1], 0, 1, 2), turn(k2, *dims), turn(v2, *dims), table,
                               starts, query=turn(new[2], 0, 1, 2), rotation=rotation_tables(n, 128))
            made.append((k2, v2, out))
        assert all(torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0)) for x, y in zip(*made))
    assert _ops.device_error() is None


@pytest.mark.parametrize('dtype', DTYPES)
def test_captured_step_of_a_cache(dtype):
    """Two layers of a decode step captured once and replayed over steps that fill and open pages, with other
    sequences admitted and released in between, beside the same steps as calls on a second cache."""
    g = gen(14)
    hq, hkv, dim, layers, batch = 8, 2, 128, 2, 3
    tables = rotation_tables(160, dim)
    caches = [PagedKVCache(60, 16, batch_capacity=5, max_length=160) for _ in range(2)]
    new = [[randn(batch, h, 1, dim, dtype=dtype, g=g) for h in (hq, hkv, hkv)] for _ in range(layers)]

    def layers_of(cache):
        out = []
        for layer, (q, k, v) in enumerate(new):
            out.append(cache.attend(cache.append(k, v, layer, query=q, rotation=tables), layer))
        return out

    def prompt(counts, first):
        for layer in range(layers):
            k, v = (randn(len(counts), hkv, max(counts), dim, dtype=dtype, g=g) for _ in range(2))
            for cache in caches:
                if layer == 0:
                    cache.begin(counts, first)
                cache.append(k, v, layer, rotation=tables)

    for cache in caches:
        cache.admit(batch)
    prompt([15, 1, 40], 0)
    captured, eager = caches
    for cache in caches:
        cache.begin()
    want = layers_of(eager)
    layers_of(captured)  # as warm-up: stores the same rows as the capture's first replay
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layers_of(captured)
        with pytest.raises(RuntimeError, match='not inside its capture'):
            captured.begin()
    for step in range(24):
        if step == 8:
            for cache in caches:
                cache.admit(2)
            prompt([20, 33], batch)
        if step == 16:
            for cache in caches:
                assert cache.release([False] * batch + [True] * 2) == [0, 1, 2]
        if step:
            for q, k, v in new:
                for t in (q, k, v):
                    t.copy_(randn(*t.shape, dtype=dtype, g=g))
            for cache in caches:
                cache.begin([1] * batch, 0)
            want = layers_of(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), step
    assert captured.lengths == eager.lengths == [39, 25, 64]
    kp, vp = captured._pools[1]
    check_attention(got[1], paged_append(new[1][1], new[1][2], kp.clone(), vp.clone(), captured.page_table(),
                                         torch.tensor([38, 24, 63], device='cuda'), query=new[1][0], rotation=tables),
                    kp, vp, captured.page_table(), captured.lengths, dim ** -0.5, 16, dtype)
    assert _ops.device_error() is None


@pytest.mark.parametrize('hq,hkv,dim,page,lengths', [
    (16, 2, 128, 16, [200, 1000, 4000]), (28, 4, 128, 64, [2500] * 9), (8, 8, 64, 32, [3000, 700, 41]),
    (4, 2, 256, 16, [3000, 500]), (32, 2, 128, 16, [9000, 300]), (6, 2, 96, 16, [1500, 90]), (8, 1, 128, 16, [130000])])
def test_attention_in_fp32_has_a_bound_of_its_own(hq, hkv, dim, page, lengths):
    """Over the outputs of a call, whose single errors are of either sign.

    Signed mean, with values above 1: an output is a mean of its values, each off by 2^-23 to either side (its
    parts), summed by blocks of 16 keys whose two large products are cut toward zero, 2^-24 of the sum each, then
    in rounded additions. So the mean over the outputs is low by 2^-23 and scatters with the rounding of single
    outputs (2^-22 each at most): 2^-23 + 2^-22 / sqrt(outputs).
    Root mean square over that of the outputs, with normal q, k, v and a scale of D^-1/2, where a score is D products
    of D^-1/2 and a weight's relative error counts as a value's does. A product of two operands in parts is off
    by 2^-21 of itself (2^-23 for each, 2^-22 dropped): 2^-21 for the score's, 2^-21 for the values'. Four
    instructions' sums are cut by 2^-23 each: 2^-21 for a score (the parts of D / 32 sums of 32, independent); two for
    the values of a block, 2^-22. The scaled score's rounding, its distance's and the exponential's: 2^-22 each.
    Together sqrt(3 2^-42 + 4 2^-44) = 2^-20."""
    g = gen(21 + dim)
    batch, scale = len(lengths), dim ** -0.5
    n = torch.tensor(lengths, device='cuda')
    for slack in (0, -(-13000 // page)):
        kp, vp, table = filled(batch, hkv, dim, page, lengths, torch.float32, g, slack=slack)
        q = randn(batch, hq, 1, dim, dtype=torch.float32, g=g)
        above = vp.abs() + 1.0
        out, low = paged_attention(q, kp, vp, table, n).double(), paged_attention(q, kp, above, table, n).double()
        own, signed = [], []
        for b, m in enumerate(lengths):
            slot = torch.arange(m, device='cuda')
            where = table[b][slot // page]
            k, v, w = (x[where, :, slot % page].transpose(0, 1).double() for x in (kp, vp, above))
            p = torch.softmax(q[b, :, 0].double().view(hkv, hq // hkv, dim) @ k.transpose(1, 2) * scale, -1)
            ref = p @ v
            own.append((out[b, 0].view_as(ref) - ref) / ref.square().mean().sqrt())
            ref = p @ w
            signed.append((low[b, 0].view_as(ref) - ref) / ref)
        own, signed = (torch.cat([x.flatten() for x in part]) for part in (own, signed))
        assert signed.mean().abs() <= 2.0 ** -23 + 2.0 ** -22 / signed.numel() ** 0.5, signed.mean().item()
        assert own.square().mean().sqrt() <= 2.0 ** -20, own.square().mean().sqrt().item()


@pytest.mark.parametrize('dim,slack', [(128, 0), (64, 900), (96, 0)])
def test_attention_keys_of_the_types_lowest_value(dim, slack):
    """fp32 keys that hold the type's lowest value, whose first part rounds to -inf, weigh nothing beside the
    others where their products are negative, and everything where they are positive."""
    g = gen(22)
    kp, vp, table = filled(1, 1, dim, 16, [300], torch.float32, g, slack=slack)
    q = torch.zeros(1, 2, 1, dim, device='cuda')
    q[0, 0, 0, 1], q[0, 1, 0, 1] = 0.25, -0.25
    kp[:, :, :, 1] = 0.0
    kp[table[0, 2], 0, 5, 1] = torch.finfo(torch.float32).min
    out = paged_attention(q, kp, vp, table, torch.tensor([300], device='cuda'), 1.0)[0, 0].double()
    slot = torch.arange(300, device='cuda')
    v = vp[table[0][slot // 16], 0, slot % 16].double()
    rest = (v.sum(0) - v[37]) / 299
    # equal weights of 1, summed exactly: the values' parts, 20 roundings of sums and one of the quotient
    assert ((out[0] - rest).abs() <= 24 * 2.0 ** -24 * v.abs().mean(0) + 2.0 ** -23 * v.abs().mean(0)).all()
    assert ((out[1] - v[37]).abs() <= 2.0 ** -22 * v[37].abs()).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim,off,slack', [(128, 0, 0), (128, 0, 900), (128, 1, 0), (96, 0, 0), (41, 0, 0)])
def test_attention_infinite_values(dtype, dim, off, slack):
    """An infinite value makes its dim of its KV head's outputs infinite or NaN, in every kernel and launch form,
    and no other; behind the length it is not there."""
    g = gen(15)
    lengths = [3000, 40, 700]
    kp, vp, table = filled(3, 2, dim, 16, lengths, dtype, g, slack=slack)
    if off:  # off 16-byte alignment
        kp, vp = (torch.zeros(p.numel() + 1, device='cuda', dtype=dtype)[1:].view(p.shape).copy_(p) for p in (kp, vp))
    q = randn(3, 8, 1, dim, dtype=dtype, g=g)
    n = torch.tensor(lengths, device='cuda')
    want = paged_attention(q, kp, vp, table, n)
    check_attention(want, q, kp, vp, table, lengths, dim ** -0.5, 16, dtype)
    vp[table[0, 9], 0, 3, 17] = math.inf
    vp[table[1, 1], 1, 2, 5] = -math.inf
    vp[table[2, 43], 1, 13, 7] = math.inf  # position 701 of 700
    out = paged_attention(q, kp, vp, table, n)
    lost = torch.zeros_like(out, dtype=torch.bool)
    lost[0, 0, :4, 17] = lost[1, 0, 4:, 5] = True
    assert torch.equal(~out.isfinite(), lost) and torch.equal(out[~lost], want[~lost])
    assert _ops.device_error() is None


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('hq,hkv,dim,page,off,slack', [
    (4, 2, 128, 16, 0, 0), (4, 2, 128, 16, 0, 900), (4, 2, 128, 24, 0, 0), (4, 2, 128, 24, 0, 600), (4, 2, 64, 16, 0, 900),
    (4, 2, 256, 16, 0, 900), (20, 1, 128, 16, 0, 900), (4, 2, 128, 16, 1, 0), (4, 2, 40, 7, 0, 0), (4, 2, 80, 16, 0, 900)])
def test_bad_pages_in_every_kernel(dtype, hq, hkv, dim, page, off, slack):
    """Pages outside the pools, inside an item of one CTA, of a cluster and of several shares: reported, and the
    outputs are those without these pages' positions, in every kernel, launch form and type."""
    g = gen(8)
    lengths = [4000, 6 * page + 3, 33]
    kp, vp, table = filled(3, hkv, dim, page, lengths, dtype, g, slack=slack)
    if off:
        kp, vp = (torch.zeros(p.numel() + 1, device='cuda', dtype=dtype)[1:].view(p.shape).copy_(p) for p in (kp, vp))
    q = randn(3, hq, 1, dim, dtype=dtype, g=g)
    for bad in (-1, kp.shape[0], 1 << 45):
        t = table.clone()
        t[0, 5], t[0, 90], t[1, 2] = bad, bad, bad
        out = paged_attention(q, kp, vp, t, torch.tensor(lengths, device='cuda'))
        err = _ops.device_error()
        assert err is not None and err[0] == 'page table'
        for b, gone in enumerate(((5, 90), (2,), ())):
            rest = [i for i in range(table.shape[1]) if i not in gone]
            check_attention(out[b:b + 1], q[b:b + 1], kp, vp, table[b:b + 1, rest], [lengths[b] - len(gone) * page],
                            dim ** -0.5, page, dtype)
    if table.shape[1] * page == lengths[0]:  # a length past the table counts to its end, one below zero not at all
        out = paged_attention(q, kp, vp, table, torch.tensor([1 << 40, lengths[1], -5], device='cuda'))
        err = _ops.device_error()
        assert err is not None and err[0] == 'page table'
        check_attention(out, q, kp, vp, table, [*lengths[:2], 0], dim ** -0.5, page, dtype)
    assert _ops.device_error() is None


@pytest.mark.parametrize('dtype,dim', [(torch.bfloat16, 128), (torch.float16, 128), (torch.float32, 64)])
def test_prompts_through_the_plain_calls(dtype, dim):
    """Prompts enter beside a live sequence: stored, queries and keys rotated by the same launch, attention of
    their own rows; then a step of one token for all."""
    from analysis_spec_b200.tree_attention import prompt_mask, tree_verify_attention
    g = gen(16)
    hq, hkv, lengths = 8, 2, [9, 33, 1]
    cache = PagedKVCache(20, 16, batch_capacity=4, max_length=80)
    tables = rotation_tables(80, dim)
    kept = []
    for group in ([20], lengths):
        first, masks = cache.admit(len(group)), {}
        cache.begin(group, first)
        q, k, v = (randn(len(group), h, max(group), dim, dtype=dtype, g=g) for h in (hq, hkv, hkv))
        qk = cache.append(k, v, 0, query=torch.cat((q, k), 1), rotation=tables)
        q, k = qk.split((hq, hkv), 1)
        out, _ = tree_verify_attention(None, q, k, v, prompt_mask(masks, q))
        for b, n in enumerate(group):
            kept.append((k[b, :, :n], v[b, :, :n]))
            kp, vp = cache._pools[0]
            slot = torch.arange(n, device='cuda')
            at = cache.page_table()[first + b][slot // 16]
            assert torch.equal(kp[at, :, slot % 16].transpose(0, 1), k[b, :, :n])
            # a row sees the rows up to itself. The verify attention holds its weights in the dtype once: each is off
            # by u of itself, in the products and not in their total, which adds 2 u max |v| to the bound above
            heads, u = torch.arange(hq, device='cuda') // (hq // hkv), torch.finfo(dtype).eps / 2
            qq, kk, vv = q[b, :, :n].double(), k[b, heads, :n].double(), v[b, heads, :n].double()
            hidden = torch.ones(n, n, dtype=torch.bool, device='cuda').triu(1)
            ref = torch.softmax((qq @ kk.transpose(1, 2) * dim ** -0.5).masked_fill(hidden, -math.inf), -1) @ vv
            ds = dim ** 0.5 * 2.0 ** -23 * (qq.abs() @ kk.abs().transpose(1, 2)).max()
            tol = u * ref.abs() + 2 * (2 * ds + u + 2.0 ** -20 + n * 2.0 ** -24) * vv.abs().amax()
            assert ((out[b, :n].transpose(0, 1).double() - ref).abs() <= tol).all()
    cache.begin()
    q, k, v = (randn(4, h, 1, dim, dtype=dtype, g=g) for h in (hq, hkv, hkv))
    q = cache.append(k, v, 0, query=q, rotation=tables)
    out = cache.attend(q, 0)
    kp, vp = cache._pools[0]
    assert cache.lengths == [21, 10, 34, 2]
    check_attention(out, q, kp, vp, cache.page_table(), cache.lengths, dim ** -0.5, 16, dtype)
    for b, (k, v) in enumerate(kept):
        slot = torch.arange(k.shape[1], device='cuda')
        at = cache.page_table()[b][slot // 16]
        assert torch.equal(kp[at, :, slot % 16].transpose(0, 1), k) and torch.equal(vp[at, :, slot % 16].transpose(0, 1), v)
    assert _ops.device_error() is None


def test_prompt_and_steps_in_either_inference_mode():
    """The transformers protocol inside and outside inference mode gives the same numbers."""
    from analysis_spec_b200.tree_attention import tree_verify_attention
    g = gen(17)
    rows = [randn(2, h, 12, 128, dtype=torch.bfloat16, g=g) for h in (8, 2, 2)]
    got = []
    for modes in ((True, False, True), (False, True, False)):
        cache, outs = PagedKVCache(12, 8, batch_capacity=2, max_length=40), []
        cache.prompt_lengths([10, 3])
        for inside, (lo, hi) in zip(modes, ((0, 10), (10, 11), (11, 12))):
            with torch.inference_mode(inside):
                q, k, v = (x[:, :, lo:hi].clone() for x in rows)
                for layer in range(2):
                    k2, v2 = cache.update(k, v, layer)
                    outs.append(tree_verify_attention(None, q, k2, v2, None)[0].clone())
        got.append(outs)
        assert cache.lengths == [12, 5]
    for x, y in zip(*got):
        assert torch.equal(x, y)
    assert _ops.device_error() is None
