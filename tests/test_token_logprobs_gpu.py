"""Log-probabilities of tokens, entropy, top alternatives and their gradient, against 64 bits.

Tolerances. With R the largest |z_i - max z| that matters (finite entries): a scaled logit's distance
to the maximum carries 2 roundings, 2^-23 R, an exponential 2^-22 of itself beside that, a sum of V
positive terms at most (V / 128 + 32) 2^-24 of itself (no thread adds more than V / 128 of them, then a
tree), so log-probabilities are off by at most
    e = 2^-21 (1 + R) + (V / 128 + 32) 2^-24,
and the entropy, a mean of distances up to R under weights that are off by e, by (1 + R) e. A gradient
entry -p (A + g (log p + H)) / T is off by p (|A| + |g| (|log p| + H + 1)) (1 + R) 3 e / T (weight,
bracket and entropy), then u |ref| for its rounding, u = eps / 2 of the dtype.
"""
import math

import pytest
import torch

from analysis_spec_b200 import _ops
from analysis_spec_b200.token_logprobs import token_logprobs
from analysis_spec_b200.tree_verification import VerifiedPath

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def bounds(z):
    """(R, e) of scaled logits z (rows, V) float64."""
    finite = z.isfinite()
    top = z.masked_fill(~finite, -math.inf).amax(-1)
    low = z.masked_fill(~finite, math.inf).amin(-1)
    r = (top - low).clamp(min=0, max=120.0).nan_to_num(0.0)  # beyond 104 an exponential is 0 in fp32
    return r, 2.0 ** -21 * (1 + r) + (z.shape[-1] / 128 + 32) * 2.0 ** -24


def order(x, k):
    x = x.double() + 0.0
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    return torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :k]


def check_forward(r, logits, tokens, top, temperature):
    z = logits.double() / temperature
    flat, tok = z.reshape(-1, z.shape[-1]), tokens.reshape(-1) if tokens is not None else None
    live = torch.ones(flat.shape[0], dtype=torch.bool, device='cuda') if tok is None else tok >= 0
    spread, e = bounds(flat)
    e = e + 2.0 ** -23 * spread  # 1 / temperature is rounded once
    lp = torch.log_softmax(flat, -1)
    entropy = torch.special.entr(lp.exp()).sum(-1)
    if tok is not None:
        want = lp.gather(1, tok.clamp(min=0)[:, None])[:, 0]
        got = r.logprobs.reshape(-1).double()
        assert not got[~live].any()
        same = (got == want) | ((got - want).abs() <= e)
        assert same[live].all(), (got - want).abs()[live].max()
    got = r.entropy.reshape(-1).double()
    assert ((got - entropy).abs() <= (1 + spread) * e)[live].all(), (got - entropy).abs()[live].max()
    if top:
        ids = order(logits.reshape(flat.shape), top)
        assert torch.equal(r.top_ids.reshape(-1, top)[live], ids[live])
        want, got = lp.gather(1, ids), r.top_logprobs.reshape(-1, top).double()
        assert ((got == want) | ((got - want).abs() <= e[:, None]))[live].all()
        assert (r.top_ids.reshape(-1, top)[~live] == -1).all() and not r.top_logprobs.reshape(-1, top)[~live].any()
    else:
        assert r.top_ids is None and r.top_logprobs is None


def some_logits(rows, vocab, dtype, g, banned=5):
    x = (3.0 * torch.randn(rows, vocab, device='cuda', generator=g)).to(dtype)
    if vocab > 50:
        x[:, torch.randint(0, vocab, (banned,), device='cuda', generator=g)] = -math.inf
    return x


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,vocab,top,temperature', [
    (1, 1, 1, 1.0), (3, 2, 2, 1.0), (5, 7, 5, 0.5), (2, 97, 32, 1.0), (7, 1000, 10, 2.0), (4, 4099, 20, 0.7),
    (1, 32000, 10, 1.0), (40, 32000, 1, 1.3), (3, 151644, 10, 1.0), (300, 8192, 5, 1.0), (2, 151643, 32, 1.0),
    (700, 513, 3, 1.0), (1, 300007, 4, 1.0), (33, 65536, 0, 1.0), (300, 151644, 10, 1.0), (100, 40000, 5, 1.0), (200, 65536, 7, 0.9)])
def test_forward(rows, vocab, top, temperature, dtype):
    g = gen(rows + vocab)
    x = some_logits(rows, vocab, dtype, g)
    tokens = torch.randint(0, vocab, (rows,), device='cuda', generator=g)
    if rows > 2:
        tokens[rows // 2] = -1
        x[rows // 2] = math.nan  # a skipped row is not read
    r = token_logprobs(x, tokens, top=top, temperature=temperature)
    check_forward(r, x, tokens, top, temperature)
    assert r.logprobs.dtype == r.entropy.dtype == torch.float32
    if top:  # without tokens
        live = torch.arange(rows, device='cuda') != rows // 2 if rows > 2 else slice(None)
        r2 = token_logprobs(x, top=top, temperature=temperature)
        assert r2.logprobs is None and torch.equal(r2.top_ids[live], r.top_ids[live])
        assert torch.equal(r2.entropy[live], r.entropy[live])
    assert _ops.device_error() is None


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('vocab', [5000, 151644])
def test_ties_and_orders(dtype, vocab):
    """Equal logits go to the lower id wherever they lie; rising, falling and constant rows."""
    g = gen(vocab)
    rows = [torch.zeros(vocab, device='cuda'), torch.arange(vocab, device='cuda') / vocab * 20,
            -torch.arange(vocab, device='cuda') / vocab * 20, torch.randint(0, 3, (vocab,), device='cuda', generator=g).float(),
            torch.where(torch.arange(vocab, device='cuda') % 2 == 0, 0.0, -0.0),
            torch.full((vocab,), -math.inf, device='cuda'), torch.full((vocab,), -math.inf, device='cuda')]
    rows[-1][vocab - 3:] = 1.0           # fewer finite entries than alternatives
    rows += [torch.full((vocab,), torch.finfo(dtype).min, device='cuda')]
    rows[-1][77] = 2.0
    x = torch.stack(rows).to(dtype)
    tokens = torch.full((len(rows),), vocab - 1, device='cuda')
    r = token_logprobs(x, tokens, top=20)
    assert torch.equal(r.top_ids, order(x, 20))
    finite = [0, 1, 2, 3, 4, 6, 7]
    sub = type(r)(*(t[finite] for t in r))
    check_forward(sub, x[finite], tokens[finite], 20, 1.0)
    assert r.logprobs[5] == -math.inf and r.entropy[5] == 0 and (r.top_logprobs[5] == -math.inf).all()
    assert r.entropy[7] == 0 and r.top_logprobs[7, 0] == 0 and r.logprobs[7] < -1e4


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('vocab', [7, 2500, 40000])
def test_rows_of_extreme_values(dtype, vocab):
    """Rows that hold only a mask's lowest value, or large equal values, are uniform; gradients too."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.full((4, vocab), low, device='cuda', dtype=dtype)
    x[1] = high
    x[2] = low / 4
    x[3, vocab // 2] = high  # the distance passes the type's range
    tokens = torch.full((4,), vocab // 2, device='cuda')
    x.requires_grad_(True)
    r = token_logprobs(x, tokens, top=3, temperature=0.5)
    e = 2.0 ** -21 + (vocab / 128 + 32) * 2.0 ** -24
    assert (r.logprobs[:3] + math.log(vocab)).abs().max() <= e * math.log(vocab) + e
    assert (r.entropy[:3] - math.log(vocab)).abs().max() <= e * math.log(vocab) + e
    assert r.logprobs[3] == 0 and r.entropy[3] == 0
    assert torch.equal(r.top_ids, order(x.detach(), 3))
    grad, = torch.autograd.grad(r.logprobs, x, torch.ones(4, device='cuda'))
    want = torch.full((4, vocab), -2.0 / vocab, device='cuda', dtype=torch.float64)
    want[:, vocab // 2] += 2.0
    want[3] = 0.0
    u = torch.finfo(dtype).eps / 2
    assert ((grad.double() - want).abs() <= (u + 4 * e) * want.abs() + 2 * e * 2 / vocab + 2.0 ** -25).all()


@pytest.mark.parametrize('dtype', DTYPES)
def test_nan_and_infinity(dtype):
    x = some_logits(4, 3000, dtype, gen(1))
    x[0, 1234] = math.nan
    x[1, 99] = math.inf
    x[3, 2999] = math.nan
    tokens = torch.tensor([5, 99, 7, -1], device='cuda')
    r = token_logprobs(x, tokens, top=4)
    assert r.logprobs[:2].isnan().all() and r.entropy[:2].isnan().all() and r.top_logprobs[:2].isnan().all()
    assert torch.equal(r.top_ids[:3], order(x[:3], 4))
    check_forward(type(r)(*(t[2:] for t in r)), x[2:].nan_to_num(0.0), tokens[2:], 4, 1.0)
    leaf = x.clone().requires_grad_(True)
    s = token_logprobs(leaf, tokens)
    grad, = torch.autograd.grad((s.logprobs, s.entropy), leaf, (torch.ones(4, device='cuda'),) * 2)
    assert grad[:2].isnan().all() and not grad[2].isnan().any() and not grad[3].any()


def test_layouts_and_row_selection():
    """(vocabulary,), (rows, vocabulary), shifted (batch, rows - 1, vocabulary) views, selected rows."""
    g = gen(2)
    base = some_logits(5 * 9, 1003, torch.bfloat16, g).view(5, 9, 1003)
    tokens = torch.randint(0, 1003, (9, 5), device='cuda', generator=g).T
    shifted = token_logprobs(base[:, :-1], tokens[:, 1:], top=3)
    check_forward(shifted, base[:, :-1], tokens[:, 1:], 3, 1.0)
    one = token_logprobs(base[2, 3], tokens[2, 4], top=3)
    assert one.logprobs.shape == () and torch.equal(one.logprobs, shifted.logprobs[2, 3])
    assert torch.equal(one.top_ids, shifted.top_ids[2, 3])
    sliced = base.flatten(0, 1)[::2, 1:500]  # a slice of the vocabulary
    t = torch.randint(0, 499, (23,), device='cuda', generator=g)
    check_forward(token_logprobs(sliced, t, top=2), sliced, t, 2, 1.0)
    same = base[:1, :1].expand(5, 9, 1003)
    check_forward(token_logprobs(same, tokens, top=1), same, tokens, 1, 1.0)
    rows = torch.randint(-1, 9, (5, 4), device='cuda', generator=g)
    chosen = torch.where(rows >= 0, torch.randint(0, 1003, (5, 4), device='cuda', generator=g), -1)
    picked = token_logprobs(base, chosen, rows=rows, top=2)
    full = base.gather(1, rows.clamp(min=0)[..., None].expand(-1, -1, 1003))
    check_forward(picked, full, chosen, 2, 1.0)
    only = token_logprobs(base, rows=rows, top=2)
    assert torch.equal(only.top_ids, picked.top_ids) and torch.equal(only.entropy, picked.entropy)
    for shape in ((0, 50), (3, 0, 50)):
        empty = token_logprobs(torch.zeros(shape, device='cuda'), torch.zeros(shape[:-1], dtype=torch.long, device='cuda'),
                               top=2)
        assert empty.logprobs.shape == shape[:-1] and empty.top_ids.shape == (*shape[:-1], 2)
    assert _ops.device_error() is None


def test_verified_path_log_probs():
    """The accepted tokens of a verify round under its logits."""
    g = gen(3)
    logits = some_logits(3 * 8, 700, torch.bfloat16, g).view(3, 8, 700)
    tokens = torch.tensor([[4, 9, -1], [600, -1, -1], [1, 2, 3]], device='cuda')
    rows = torch.tensor([[0, 5, -1], [0, -1, -1], [0, 2, 7]], device='cuda')
    path = VerifiedPath(tokens, rows, rows, (tokens >= 0).sum(1))
    r = path.log_probs(logits, top=2, temperature=0.9)
    full = logits.gather(1, rows.clamp(min=0)[..., None].expand(-1, -1, 700))
    check_forward(r, full, tokens, 2, 0.9)


def test_out_of_range_is_reported_and_skipped():
    x = some_logits(3, 200, torch.float32, gen(4))
    r = token_logprobs(x, torch.tensor([5, 200, 7], device='cuda'), top=1)
    assert _ops.device_error() == ('token index', 200)
    assert r.logprobs[1] == 0 and r.entropy[1] == 0 and r.top_ids[1, 0] == -1 and r.top_ids[2, 0] >= 0
    r = token_logprobs(x[None], rows=torch.tensor([[0, 3, 1 << 40]], device='cuda'), top=1)
    assert _ops.device_error()[0] == 'token index'
    assert r.top_ids[0, 1, 0] == -1 and r.top_ids[0, 0, 0] >= 0
    leaf = x.clone().requires_grad_(True)
    s = token_logprobs(leaf, torch.tensor([5, 200, 7], device='cuda'))
    s.logprobs.sum().backward()
    assert _ops.device_error() == ('token index', 200) and not leaf.grad[1].any() and leaf.grad[0].any()


# ---- gradient ----------------------------------------------------------------------------------

def reference_grad(logits, tokens, top_ids, temperature, ga, gh, gt):
    """The formula in 64 bits and its error bound's scale."""
    z = logits.double() / temperature
    lp = torch.log_softmax(z, -1)
    p = lp.exp()
    live = torch.ones(len(z), 1, device='cuda') if tokens is None else (tokens >= 0)[:, None].double()
    finite = torch.where(p > 0, lp, 0.0)
    entropy = -(p * finite).sum(-1, keepdim=True)
    a = torch.zeros_like(live) if ga is None else ga.double()[:, None]
    h = torch.zeros_like(live) if gh is None else gh.double()[:, None]
    every = a.clone()
    d = torch.zeros_like(z)
    if ga is not None:
        d.scatter_add_(1, tokens.clamp(min=0)[:, None], a)
    if gt is not None:
        every = every + gt.double().sum(-1, keepdim=True)
        d.scatter_add_(1, top_ids.clamp(min=0), gt.double())
    d = (d - p * (every + h * (finite + entropy))) * live / temperature
    mass = a.abs() if gt is None else a.abs() + gt.double().abs().sum(-1, keepdim=True)
    size = p * (mass + h.abs() * (finite.abs() + entropy + 1)) / temperature
    return d, size


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,vocab,top,temperature', [
    (1, 1, 1, 1.0), (3, 5, 2, 0.5), (2, 1000, 32, 1.0), (6, 4099, 5, 1.4), (40, 32000, 0, 1.0), (2, 151644, 10, 0.8),
    (200, 777, 1, 1.0)])
def test_gradient_against_the_formula(rows, vocab, top, temperature, dtype):
    g = gen(rows * 3 + vocab)
    x = some_logits(rows, vocab, dtype, g)
    tokens = torch.randint(0, vocab, (rows,), device='cuda', generator=g)
    if rows > 2:
        tokens[1] = -1
        x[1] = math.nan
    if top:
        tokens[0] = order(x[:1], 1)[0, 0]  # the token is one of its row's alternatives
    leaf = x.clone().requires_grad_(True)
    ga, gh = (torch.randn(rows, device='cuda', generator=g) for _ in range(2))
    gt = torch.randn(rows, top, device='cuda', generator=g) if top else None
    clean = torch.where(x.isnan(), torch.zeros_like(x), x)
    z = clean.double() / temperature
    spread, e = bounds(z)
    for parts in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
        use = [v if on else None for v, on in zip((ga, gh, gt), parts)]
        if all(v is None for v in use):
            continue
        r = token_logprobs(leaf, tokens, top=top, temperature=temperature)
        outs = [o for o, v in zip((r.logprobs, r.entropy, r.top_logprobs), use) if v is not None]
        got, = torch.autograd.grad(outs, leaf, [v for v in use if v is not None])
        ref, size = reference_grad(clean, tokens, r.top_ids, temperature, *use)
        assert got.dtype == dtype and got.is_contiguous()
        u = torch.finfo(dtype).eps / 2
        small = 2.0 ** -25 if dtype == torch.float16 else 1e-38
        # the special entries add their own gradient to -p (...): one fp32 rounding of its size
        tol = u * ref.abs() * 1.01 + size * ((1 + spread) * 3 * e)[:, None] + 2.0 ** -22 * (ref.abs() + size) + small
        bad = (got.double() - ref).abs() > tol
        assert not bad.any(), (parts, bad.sum().item(), (got.double() - ref).abs().max().item())
    assert _ops.device_error() is None


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('vocab,pitch', [(31, 33), (501, 501), (4099, 4100), (9001, 9015)])
def test_gradient_of_views_at_any_offset(vocab, pitch, dtype):
    """Logits whose entries lie 0 to 16 entries off the gradient's, words across each other included; the
    entries around the view are NaN."""
    g = gen(vocab)
    tokens = torch.randint(0, vocab, (3,), device='cuda', generator=g)
    ga, gh = (torch.randn(3, device='cuda', generator=g) for _ in range(2))
    u = torch.finfo(dtype).eps / 2
    small = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    for offset in (0, 1, 2, 3, 7, 8, 15, 16):
        store = torch.full((3 * pitch + 32,), math.nan, dtype=dtype, device='cuda')
        x = store[offset:offset + 3 * pitch].view(3, pitch)[:, :vocab]
        x.copy_(some_logits(3, vocab, dtype, g))
        leaf = x.detach().requires_grad_(True)
        assert leaf.data_ptr() == x.data_ptr()
        r = token_logprobs(leaf, tokens, temperature=0.9)
        got, = torch.autograd.grad((r.logprobs, r.entropy), leaf, (ga, gh))
        z = x.double() / 0.9
        spread, e = bounds(z)
        ref, size = reference_grad(x, tokens, None, 0.9, ga, gh, None)
        tol = u * ref.abs() * 1.01 + size * ((1 + spread) * 3 * e)[:, None] + 2.0 ** -22 * (ref.abs() + size) + small
        assert ((got.double() - ref).abs() <= tol).all(), (offset, (got.double() - ref).abs().max().item())
    assert _ops.device_error() is None


def test_gradient_against_differences():
    """Central differences of the kernel's own outputs in fp32: with a step of h the quotient is off by
    h^2 / 6 of a third derivative (at most 1 for log-probabilities, 1 + R for the entropy) and by the
    outputs' own error, (1 + R) e / h."""
    g = gen(5)
    x = torch.randn(1, 12, device='cuda', generator=g)
    tokens = torch.tensor([4], device='cuda')
    h, weights = 2.0 ** -5, (0.7, -1.3)
    spread, e = bounds(x.double())

    def value(v):
        r = token_logprobs(v, tokens.expand(v.shape[0]))
        return weights[0] * r.logprobs + weights[1] * r.entropy

    leaf = x.clone().requires_grad_(True)
    grad, = torch.autograd.grad(value(leaf).sum(), leaf)
    step = h * torch.eye(12, device='cuda')
    slope = (value(x + step) - value(x - step)) / (2 * h)
    tol = (sum(map(abs, weights)) * (1 + spread) * (h * h / 6 * 2 + 2 * e / h)).item()
    assert (grad[0] - slope).abs().max() <= tol


def test_gradient_layouts_streams_and_graphs():
    """Shifted and broadcast leaves, expanded gradients, another stream; a backward pass captured into
    a graph and replayed on changed logits (nothing eager of the same leaf is alive)."""
    g = gen(6)
    base = some_logits(4 * 6, 501, torch.float32, g, banned=0).view(4, 6, 501).requires_grad_(True)
    tokens = torch.randint(0, 501, (4, 6), device='cuda', generator=g)

    def loss(v, t):
        r = token_logprobs(v, t, temperature=1.5)
        return r.logprobs.sum() - 0.1 * r.entropy.mean()  # expanded gradients

    def plain(v, t):
        lp = torch.log_softmax(v.double() / 1.5, -1)
        return lp.gather(-1, t[..., None]).sum() - 0.1 * torch.special.entr(lp.exp()).sum(-1).mean()

    for view in (lambda v: v, lambda v: v[:, :-1], lambda v: v[:1].expand(4, 6, 501), lambda v: v[:, ::2, 3:]):
        t = tokens[:, :view(base).shape[1]] % view(base).shape[2]
        got, = torch.autograd.grad(loss(view(base), t), base)
        want, = torch.autograd.grad(plain(view(base), t), base)
        assert (got - want).abs().max() <= 4e-5 * want.abs().max()  # e of the forward at R < 32, four rows summed
    want, = torch.autograd.grad(plain(base, tokens), base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, = torch.autograd.grad(loss(base, tokens), base)
    torch.cuda.synchronize()
    assert (got - want).abs().max() <= 4e-5 * want.abs().max()
    del got, want
    static = base.detach().clone().requires_grad_(True)
    with torch.cuda.stream(side):  # warm up on the capture's kind of stream
        torch.autograd.grad(loss(static, tokens), static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, = torch.autograd.grad(loss(static, tokens), static)
    for scale in (1.0, 0.3):
        with torch.no_grad():
            static.copy_(base * scale)
        graph.replay()
        torch.cuda.synchronize()
        fresh = (base.detach() * scale).requires_grad_(True)
        want, = torch.autograd.grad(plain(fresh, tokens), fresh)
        assert (out - want).abs().max() <= 4e-5 * want.abs().max()


def test_twice_differentiated_is_refused():
    x = torch.randn(2, 30, device='cuda', requires_grad=True)
    r = token_logprobs(x, torch.tensor([1, 2], device='cuda'))
    grad, = torch.autograd.grad(r.logprobs.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='not twice differentiable'):
        torch.autograd.grad(grad.square().sum(), x)
    r = token_logprobs(x, torch.tensor([1, 2], device='cuda'), top=3)
    assert r.top_ids.grad_fn is None and not r.top_ids.requires_grad and r.top_logprobs.requires_grad
    with torch.no_grad():
        assert not token_logprobs(x, top=1).entropy.requires_grad
    y = x * 1.0
    r = token_logprobs(y, torch.tensor([1, 2], device='cuda'))
    y.add_(1.0)  # the saved logits changed
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        r.entropy.sum().backward()


def test_rows_beyond_32_bit_offsets():
    x = torch.zeros(15000, 151644, device='cuda', dtype=torch.bfloat16)  # 2.27e9 entries
    x[14999, 151640] = 9.0
    tokens = torch.full((15000,), -1, device='cuda')
    tokens[14999] = 151640
    x.requires_grad_(True)
    r = token_logprobs(x, tokens, top=1)
    assert r.top_ids[14999, 0] == 151640
    grad, = torch.autograd.grad(r.logprobs, x, torch.ones(15000, device='cuda'))
    assert grad[14999, 151640] > 0 and (grad[14999] != 0).all() and not grad[:14999].any()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('temperature', [1e-29, 1e-20, 1e-9, 1e9, 1e29])
@pytest.mark.parametrize('vocab', [7, 2500, 40000, 151644])
def test_masked_rows_at_extreme_temperatures(dtype, temperature, vocab):
    """Rows that leave five tokens, at the temperatures' ends: the equal largest share the weight (all of
    the finite ones at high temperatures), whatever the threads that meet -inf alone would make of it."""
    x = torch.full((2, vocab), -math.inf, dtype=dtype, device='cuda')
    at = torch.linspace(1, vocab - 1, 5, device='cuda').long()
    x[:, at] = 1.5
    x[1, at[1]] = 0.5 if temperature < 1 else 1.25
    tokens = torch.stack((at[0], at[4]))
    r = token_logprobs(x, tokens, top=2, temperature=temperature)
    check_forward(r, x, tokens, 2, temperature)
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, tokens, temperature=temperature)
    gh = torch.tensor([1.0, -2.0], device='cuda')
    # equal weights: the entropy's gradient -p (log p + H) / T is 0 but for the statistics' own error, 3 e p / T
    grad, = torch.autograd.grad(r.entropy, leaf, gh)
    spread, e = bounds(x.double() / temperature)
    p = torch.softmax(x.double() / temperature, -1)
    lp = torch.where(p > 0, p.log(), 0.0)
    ref = -p * (lp - (p * lp).sum(-1, keepdim=True)) * gh[:, None] / temperature
    size = p * (lp.abs() + 3) * gh.abs()[:, None] / temperature
    tol = size * ((1 + spread) * 3 * e)[:, None] + torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -25
    # 1 / T passes fp16's range, and so may a true value of ref +- tol: such ones round to infinity
    got = grad.double().clamp(torch.finfo(dtype).min, torch.finfo(dtype).max)
    assert ((got - ref).abs() <= tol).all()


@pytest.mark.parametrize('rows,vocab', [(300, 4096), (300, 70000), (2, 5000)])
def test_references_that_pass_the_fused_products_border(rows, vocab):
    """Scaled logits around +-2^20: a thread's reference changes between the form that takes the difference
    first and the fused one, by steps of log2(e) / 16 whose rounding (2^-5 at most) differs each time."""
    border = round(2.0 ** 20 * math.log(2.0) * 16) / 16
    tokens = torch.arange(rows, device='cuda') % 7
    half = torch.arange(vocab, device='cuda') * 2 >= vocab
    one = torch.arange(vocab, device='cuda') == vocab - 9
    j = torch.arange(rows, device='cuda')[:, None] % 24
    # low entries first, below -2^20; then half of the row, up to 1.6 above them and past the border
    x = torch.where(half, -border + (1 + j % 9) / 16, -border - (1 + j % 16) / 16).float()
    check_forward(token_logprobs(x, tokens, top=1), x, tokens, 1, 1.0)
    # ... and one entry past 2^20, far enough above the rest for a new reference (10 in powers of two)
    x = torch.where(one, border + (1 + j % 9) / 16, border - 7.0 - (1 + j % 16) / 16).float()
    check_forward(token_logprobs(x, tokens, top=1), x, tokens, 1, 1.0)


def test_capture_beside_a_live_eager_graph_is_refused():
    """Before anything is launched; two calls of one capture are no such case, nor is a call without a gradient."""
    g = gen(7)
    x = some_logits(3, 501, torch.float32, g).requires_grad_(True)
    tokens = torch.randint(0, 501, (3,), device='cuda', generator=g)
    want = token_logprobs(x, tokens).logprobs  # alive, on the default stream
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match='still alive'):
            token_logprobs(x, tokens)
        with torch.no_grad():
            plain = token_logprobs(x, tokens).logprobs
        other = token_logprobs(x.detach().requires_grad_(True), tokens).logprobs.detach()
    graph.replay()
    torch.cuda.synchronize()
    want = want.detach()  # its graph is gone
    assert torch.equal(plain, want) and torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first, second = token_logprobs(x, tokens), token_logprobs(x, tokens, temperature=2.0)
        grad, = torch.autograd.grad(first.logprobs.sum() + second.entropy.sum(), x)
        first, second = first.logprobs.detach(), second.entropy.detach()
    graph.replay()
    torch.cuda.synchronize()
    r, s = token_logprobs(x, tokens), token_logprobs(x, tokens, temperature=2.0)
    again, = torch.autograd.grad(r.logprobs.sum() + s.entropy.sum(), x)
    assert torch.equal(first, r.logprobs) and torch.equal(second, s.entropy) and torch.equal(grad, again)
