"""The operators over large item vocabularies against plain restatements in 64 bits.

Tolerances are bounds by arithmetic, element by element.  u = 2^-24 is half a step of 32 bits; a store to type t adds at most
finfo(t).eps / 2 of the value (or half the smallest subnormal).  The sum of a row's V exponentials is formed by at least 64 threads
one element after the other and then over at most 64 + 16 partial sums, and each online rescaling repeats an exponential: with A the
largest |z - m| log2(e) / T in the row, an exponential is off by (4 + 3 A) u (the difference, the product, the constant, 2 u of the
hardware exp2), and S and every q by E = (4 + 3 A + 2 (V / 64 + 96)) u of their value."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ALL = [F32, BF16, F16]


def stored(ref, dtype):
    """The most that one store of ``ref`` to ``dtype`` can be off (with the rounding to 32 bits in front of it)."""
    f = torch.finfo(dtype)
    return ref.abs() * (f.eps / 2 * (1 + U) + (0 if dtype == F32 else U)) + f.smallest_normal * f.eps / 2


def within(got, ref, tol):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape
    odd = ~torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got[odd & ~torch.isnan(ref)], ref[odd & ~torch.isnan(ref)])
    off = torch.where(odd, 0.0, (got - ref).abs() - tol)
    assert off.numel() == 0 or off.max() <= 0, f"off by {off.max().item():.3g} more than the bound, at {off.argmax().item()}"


def gen(seed, dev):
    return torch.Generator(device=dev).manual_seed(seed)


# ---- table rows --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,rows,d", [(1, 1, 1), (5, 3, 7), (32, 1000, 64), (257, 33, 65), (1000, 4097, 128), (63, 100, 1000), (4099, 50, 8)])
def test_embedding(rbg, cuda, dtype, n, rows, d):
    g = gen(n + d, cuda)
    table = torch.randn(rows, d, generator=g, device=cuda).to(dtype)
    ids = torch.randint(-2, rows + 2, (n,), generator=g, device=cuda)
    ids[0] = rows - 1
    there = (ids >= 0) & (ids < rows)
    for scale in (1.0, math.sqrt(d) * 1.1):
        out = rbg.embedding(table, ids, scale=scale, padding_idx=0)
        ref = table[torch.where(there, ids, 0)].double() * scale * there[:, None]
        within(out, ref, stored(ref, dtype) + 2 * U * ref.abs())  # (the scale itself is rounded to 32 bits)
        assert torch.all(out[~there] == 0)
    assert torch.equal(rbg.embedding(table, ids)[there], table[ids[there]])  # scale 1 copies


@pytest.mark.parametrize("dtype", ALL)
def test_embedding_layouts(rbg, cuda, dtype):
    g = gen(3, cuda)
    wide = torch.randn(50, 200, generator=g, device=cuda).to(dtype)
    ids = torch.randint(50, (3, 5, 7), generator=g, device=cuda)
    for table in (wide[:, 3:67], wide[:, 8:72], wide[5:, :64], wide.t()[:64].t(), wide[:, :64].t().contiguous().t(), wide[::2, 1:65], wide[:1].expand(50, 200)):
        own = ids % table.shape[0]
        assert torch.equal(rbg.embedding(table, own), table[own])
        assert torch.equal(rbg.embedding(table, own.int()), table[own])
        assert torch.equal(rbg.embedding(table, own.permute(2, 0, 1)), table[own.permute(2, 0, 1)])
    assert rbg.embedding(wide, ids[:0]).shape == (0, 5, 7, 200)
    assert torch.all(rbg.embedding(wide[:0], ids) == 0)


def runs_reference(grad, ids, rows, scale, padding):
    """(sum, sum of magnitudes, count) per row in 64 bits."""
    ok = (ids >= 0) & (ids < rows) & (ids != padding)
    g = grad.double()[ok] * scale
    zero = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device=grad.device)
    return (zero.index_add(0, ids[ok], g), zero.index_add(0, ids[ok], g.abs()),
            torch.bincount(ids[ok], minlength=rows)[:, None].double())


GRAD_SHAPES = [(1, 1, 1), (2, 5, 64), (7, 3, 65), (100, 700, 64), (255, 3, 40), (256, 1000, 513), (257, 1000, 16), (300, 50, 64), (5000, 40, 128), (6144, 40982, 64), (4096, 1, 32), (16384, 1000, 32), (16385, 511, 24),
               (16385, 512, 8), (20000, 70000, 64), (40000, 3, 100), (50000, 300000, 16), (70001, 100, 1), (33000, 1, 4), (65536, 140000, 3), (65537, 777, 4), (131072, 300, 2), (150000, 600000, 2), (1000, 20, 1024), (3000, 7, 2051)]


@pytest.mark.parametrize("n,rows,d", GRAD_SHAPES)
@pytest.mark.parametrize("dtype", ALL)
def test_embedding_grad(rbg, cuda, dtype, n, rows, d):
    g = gen(n + rows, cuda)
    grad = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    u = torch.rand(n, generator=g, device=cuda)
    ids = (rows * u * u * u).long().clamp_(max=rows - 1)
    ids[torch.rand(n, generator=g, device=cuda) < 0.05] = -1
    ids[n // 2:n // 2 + 1] = rows  # out of range
    for padding, out_dtype in ((None, None), (0, F32)):
        got = rbg.embedding_grad(grad, ids, rows, scale=1.7, padding_idx=padding, out_dtype=out_dtype)
        assert got.dtype == (out_dtype or dtype)
        ref, mag, cnt = runs_reference(grad, ids, rows, 1.7, -1 if padding is None else padding)
        within(got, ref, stored(ref, got.dtype) + mag * U * (cnt + 4))  # cnt additions in some order, the scale, its rounding
        assert torch.all(got[cnt[:, 0] == 0] == 0)
        assert torch.equal(got, rbg.embedding_grad(grad, ids, rows, scale=1.7, padding_idx=padding, out_dtype=out_dtype))


@pytest.mark.parametrize("n", [0, 1, 9, 256, 257, 3000, 20000])
def test_embedding_grad_of_nothing_and_of_one_row(rbg, cuda, n):
    grad = torch.ones(n, 64, device=cuda)
    none = torch.full((n,), -1, device=cuda)
    assert torch.all(rbg.embedding_grad(grad, none, 300) == 0)
    assert torch.all(rbg.embedding_grad(grad, torch.full_like(none, 299), 300)[299] == n)  # whole numbers below 2^24: exact in any order
    assert torch.all(rbg.embedding_grad(grad, torch.full_like(none, 7), 300, padding_idx=7) == 0)
    last = rbg.embedding_grad(grad, torch.arange(n, device=cuda) % 300, 300)
    assert torch.equal(last[:, 0], torch.bincount(torch.arange(n, device=cuda) % 300, minlength=300).float())


def test_embedding_grad_sums_in_ascending_order(rbg, cuda):
    """Within a chunk places are added one after the other in their order: 2^24 + 1 + 1 - 2^24 shows it (1 + 1 first would give 2)."""
    grad = torch.tensor([2.0 ** 24, 1.0, 1.0, -2.0 ** 24], device=cuda)[:, None].repeat(1, 4)
    ids = torch.zeros(4, dtype=torch.int64, device=cuda)
    assert torch.all(rbg.embedding_grad(grad, ids, 1) == 0.0)
    order = torch.tensor([1, 2, 0, 3], device=cuda)
    assert torch.all(rbg.embedding_grad(grad[order], ids, 1) == 2.0)


@pytest.mark.parametrize("dtype", ALL)
def test_embedding_grad_layouts(rbg, cuda, dtype):
    g = gen(5, cuda)
    wide = torch.randn(400, 200, generator=g, device=cuda).to(dtype)
    ids = torch.randint(30, (400,), generator=g, device=cuda)
    for grad in (wide[:, 3:67], wide[:, 8:72], wide[:, ::2], wide[:1].expand(400, 200)):
        assert torch.equal(rbg.embedding_grad(grad, ids, 30), rbg.embedding_grad(grad.contiguous(), ids, 30))
    three = rbg.embedding_grad(wide.view(8, 50, 200), ids.view(8, 50), 30)
    assert torch.equal(three, rbg.embedding_grad(wide, ids, 30))


def test_embedding_autograd(rbg, cuda):
    g = gen(6, cuda)
    table = torch.randn(20, 12, generator=g, device=cuda, requires_grad=True)
    ids = torch.randint(20, (4, 9), generator=g, device=cuda)
    w = torch.randn(4, 9, 12, generator=g, device=cuda)
    (rbg.embedding(table, ids, scale=0.5, padding_idx=3) * w).sum().backward()
    ref, mag, cnt = runs_reference(w.view(-1, 12), ids.view(-1), 20, 0.5, 3)
    within(table.grad, ref, stored(ref, F32) + mag * U * (cnt + 4))
    # differences: the sum is linear in the table, so a step of 1 is exact up to the roundings of two sums of 432 terms
    t = table.detach().clone()
    i = int(ids[0, 0]) if int(ids[0, 0]) != 3 else int(ids[0, 1])
    lo = (rbg.embedding(t, ids, scale=0.5).double() * w.double()).sum()
    t[i, 5] += 1.0
    hi = (rbg.embedding(t, ids, scale=0.5).double() * w.double()).sum()
    assert abs((hi - lo) - table.grad[i, 5].double()) <= 36 * 4 * U * float(w.abs().max()) * 8


def test_embedding_beyond_32_bits(rbg, cuda):
    rows, d = (1 << 25) + 11, 64  # 2^31 + 704 elements
    table = torch.zeros(rows, d, dtype=BF16, device=cuda)
    table[-1] = 3.0
    table[(1 << 25) - 1] = 2.0
    ids = torch.tensor([rows - 1, (1 << 25) - 1, rows, 5], device=cuda)
    out = rbg.embedding(table, ids)
    assert [float(v) for v in out[:, 63]] == [3.0, 2.0, 0.0, 0.0]
    del table
    grad = rbg.embedding_grad(torch.ones(4, d, dtype=BF16, device=cuda), ids, rows)
    assert torch.all(grad[-1] == 1) and torch.all(grad[(1 << 25) - 1] == 1) and torch.all(grad[5] == 1)
    assert float(grad.sum(dtype=F32)) == 3 * d


# ---- distillation ------------------------------------------------------------------------------------------------------

def distill_reference(z, idx, val, temp, w):
    """(loss, its bound, gradient, its bound) in 64 bits."""
    n, v = z.shape
    z = z.double()
    there = (idx >= 0) & (idx < v)
    at = torch.where(there, idx, 0)
    val = torch.where(there, val.double(), -math.inf)
    some = there & ~torch.isneginf(val)
    m = z.amax(1, keepdim=True)
    empty = ~some.any(1) | torch.isneginf(m[:, 0])
    p = torch.softmax(val / temp, 1)
    logq = torch.log_softmax(z / temp, 1)
    terms = torch.where(there & (p > 0), torch.xlogy(p, p) - p * logq.gather(1, at), torch.where(torch.isnan(p), p, 0.0))
    loss = torch.where(empty, 0.0, temp * temp * terms.sum(1))
    grad = logq.exp().scatter_add(1, at, torch.where(there, -p, 0.0))
    grad = torch.where(empty[:, None], 0.0, grad * (w[:, None] * temp))
    k = idx.shape[1]
    fin = torch.where(torch.isfinite(z), z, m)
    far = ((m - fin) * (1.4427 / temp)).amax(1, keepdim=True).clamp(max=160.0)  # below 2^-150 an exponential is 0 either way
    e = (4 + 3 * far + 2 * (v / 64 + 96)) * U
    tfar = torch.where(some, (val.amax(1, keepdim=True) - val) * (1.4427 / temp), 0.0).clamp(max=160.0)
    ep = (6 + 3 * tfar + k + 8) * U
    lq = torch.where(some, logq.gather(1, at), 0.0)
    lp = torch.where(some & (p > 0), torch.log(p), 0.0)
    tl = (p * (e + ep + 6 * U * (lq.abs() + lp.abs()) + (lq - lp).abs() * (ep + (k + 4) * U))).sum(1) * temp * temp + 1e-37
    q = logq.exp()
    tg = (w[:, None].abs() * temp) * (q * (e + 4 * U) + q.new_zeros(n, v).scatter_add(1, at, torch.where(some, p * (ep + 4 * U), 0.0)))
    tg = tg + (w[:, None].abs() * temp + 1) * 2.0 ** -125 + stored(grad, F32)
    return loss, torch.nan_to_num(tl, nan=0.0, posinf=0.0), grad, torch.nan_to_num(tg, nan=0.0)


def distill_inputs(seed, n, v, k, dtype, dev, pad=0):
    g = gen(seed, dev)
    z = (2 * torch.randn(n, v + pad, generator=g, device=dev)).to(dtype)[:, :v]
    idx = torch.randint(v, (n, k), generator=g, device=dev)
    val = 2 * torch.randn(n, k, generator=g, device=dev) + 3
    left = torch.randint(0, 2 * k + 1, (n, 1), generator=g, device=dev)
    none = torch.arange(k, device=dev)[None] >= left
    idx[none] = -1
    val[none] = math.nan  # whatever stands beside a missing entry
    return z, idx, val, torch.rand(n, generator=g, device=dev) + 0.5


def distill_check(rbg, z, idx, val, temp, w):
    loss, tl, grad, tg = distill_reference(z, idx, val, temp, w)
    got, gg = rbg.distill_topk_grad(z, idx, val, temperature=temp, row_weight=w)
    within(got, loss, tl)
    within(gg, grad, tg + stored(grad, z.dtype))
    assert torch.equal(rbg.distill_topk(z, idx, val, temperature=temp).isnan(), loss.isnan())
    within(rbg.distill_topk(z, idx, val, temperature=temp), loss, tl)
    leaf = z.detach().clone().requires_grad_()
    out = rbg.distill_topk(leaf, idx, val, temperature=temp)
    out.backward(w)
    within(out.detach(), loss, tl)
    within(leaf.grad, grad, tg + stored(grad, z.dtype))
    again, g2 = rbg.distill_topk_grad(z, idx, val, temperature=temp, row_weight=w)
    assert torch.equal(torch.nan_to_num(again), torch.nan_to_num(got)) and torch.equal(torch.nan_to_num(g2), torch.nan_to_num(gg))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (64, 1683, 10), (17, 1024, 256), (600, 63, 4), (2, 50001, 33), (100, 16390, 5), (513, 4099, 12),
                                   (1, 300007, 64)])
def test_distill(rbg, cuda, dtype, n, v, k):
    z, idx, val, w = distill_inputs(n + v, n, v, k, dtype, cuda)
    distill_check(rbg, z, idx, val, 2.0, w)


@pytest.mark.parametrize("dtype,v", [(F32, 12289), (F32, 20001), (F32, 30000), (F32, 40982), (F32, 60001), (F32, 65539), (F32, 70001), (BF16, 33000), (BF16, 40982),
                                     (F16, 65530), (BF16, 90001), (F16, 131077)])
def test_distill_every_row_length(rbg, cuda, dtype, v):
    """Enough rows that each has a workgroup of its own: every size of register-resident row, and the longer ones."""
    z, idx, val, w = distill_inputs(v, 512, v, 20, dtype, cuda)
    distill_check(rbg, z, idx, val, 1.0, w)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", [6, 520])
@pytest.mark.parametrize("v", [40, 9001, 40000])
def test_distill_masks(rbg, cuda, dtype, n, v):
    z, idx, val, w = distill_inputs(7, n, v, 6, dtype, cuda, pad=5)
    idx[:6], val[:6] = torch.arange(6, device=cuda) * 5, 1.0
    low = torch.finfo(dtype).min
    idx[0] = -1                                   # no entry
    val[1] = -math.inf                            # entries without weight
    z[2] = -math.inf                              # no logits
    z[3] = low                                    # all masked by the lowest value: a uniform row
    z[4, ::2] = -math.inf                         # masked items, entries 0, 10, 20 among them: an infinite loss
    z[5, 1::2], idx[5, 3:] = low, 10              # masked items, and one index four times (10 and 10, 10, 10)
    z[5, 10], val[5] = 1.0, torch.tensor([0.5, 1.0, 1.5, -math.inf, 2.0, 2.5], device=cuda)
    distill_check(rbg, z, idx, val, 1.5, w)
    loss, grad = rbg.distill_topk_grad(z, idx, val, temperature=1.5)
    assert torch.all(loss[:3] == 0) and torch.all(grad[:3] == 0) and float(loss[4]) == math.inf
    bad = z.clone()
    bad[0, 3], bad[3, 0], bad[1, 0], bad[5, 7] = math.nan, math.nan, math.inf, math.inf
    loss, grad = rbg.distill_topk_grad(bad, idx, val, temperature=1.5)
    assert torch.all(loss[:2] == 0) and torch.all(grad[:2] == 0) and torch.all(loss[3:6:2].isnan()) and torch.all(grad[3].isnan())
    # a row spoils itself alone (the same bits, from rows of the same layout: where a row starts decides which thread adds what)
    assert torch.equal(grad[6:], rbg.distill_topk_grad(z.clone(), idx, val, temperature=1.5)[1][6:])


def test_distill_differences(rbg, cuda):
    """Central differences with h = 2^-5: off by h^2 / 6 times the third derivative (at most T = 1 here) and by the losses' own bound / h."""
    z, idx, val, _ = distill_inputs(11, 4, 9, 3, F32, cuda)
    idx[:, 0], val[:, 0] = 4, 1.0
    w = torch.ones(4, device=cuda)
    _, tl, _, _ = distill_reference(z, idx, val, 1.0, w)
    _, grad = rbg.distill_topk_grad(z, idx, val)
    h = 2.0 ** -5
    for j in range(9):
        zp, zm = z.clone(), z.clone()
        zp[:, j] += h
        zm[:, j] -= h
        diff = (rbg.distill_topk(zp, idx, val).double() - rbg.distill_topk(zm, idx, val).double()) / ((zp - zm)[:, j].double())
        assert torch.all((diff - grad[:, j].double()).abs() <= h * h / 6 + 4 * tl / h + 2.0 ** -20)


@pytest.mark.parametrize("n,v", [(3, 50000), (520, 777), (520, 70001)])
def test_distill_in_place(rbg, cuda, n, v):
    z, idx, val, w = distill_inputs(2, n, v, 9, F32, cuda)
    loss, grad = rbg.distill_topk_grad(z, idx, val, row_weight=w)
    lib, b = rbg._lib.lib, ctypes.c_int64()
    rbg._lib.check(lib.rbg_distill_topk_workspace(n, v, ctypes.byref(b)))
    work = torch.empty(b.value, dtype=torch.uint8, device=cuda)
    out = torch.empty_like(loss)
    rbg._lib.check(lib.rbg_distill_topk(z.data_ptr(), v, 0, n, v, idx.data_ptr(), val.data_ptr(), 9, 1.0, w.data_ptr(), out.data_ptr(), None,
                                        z.data_ptr(), v, work.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(z, grad) and torch.equal(out, loss)


def test_distill_rows_beyond_32_bits(rbg, cuda):
    n, v = 2051, (1 << 20) + 1  # 2^31 + 3 M elements
    z = torch.zeros(n, v, dtype=BF16, device=cuda)
    z[-1, -1] = 8.0
    idx = torch.full((n, 1), v - 1, device=cuda)
    val = torch.zeros(n, 1, device=cuda)
    loss, grad = rbg.distill_topk_grad(z, idx, val)
    ref = math.log((v - 1) * math.exp(-8.0) + 1.0)
    assert abs(float(loss[-1]) - ref) < ref * 1e-3 and abs(float(loss[0]) - math.log(v)) < 1e-3
    q = math.exp(-ref)
    assert abs(float(grad[-1, -1]) - (q - 1)) < 2.0 ** -8 and abs(float(grad[-1, 0]) - math.exp(-8.0 - ref)) < 2.0 ** -8 * math.exp(-8.0 - ref)
    assert abs(float(grad[-2, -1]) - (1.0 / v - 1)) < 2.0 ** -8


# ---- log-probabilities and the preference loss -----------------------------------------------------------------------------

def logp_reference(z, y):
    """(logp, its bound, softmax, E) in 64 bits; 0 for rows without a target or without logits."""
    v = z.shape[1]
    z = z.double()
    m = z.amax(1, keepdim=True)
    there = (y >= 0) & (y < v) & ~torch.isneginf(m[:, 0])
    lq = torch.log_softmax(z, 1)
    lp = torch.where(there, lq.gather(1, torch.where(there, y, 0)[:, None])[:, 0], 0.0)
    fin = torch.where(torch.isfinite(z), z, m)
    far = ((m - fin) * 1.4427).amax(1).clamp(max=160.0)
    e = torch.nan_to_num((4 + 3 * far + 2 * (v / 64 + 96)) * U, nan=0.0)
    return lp, e + 2 * U * torch.nan_to_num(lp.abs(), posinf=0.0), lq.exp(), e, there


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m,v", [(1, 1), (3, 2), (40, 1683), (7, 60001), (600, 1025), (530, 9000), (2, 262147)])
def test_token_logp(rbg, cuda, dtype, m, v):
    g = gen(m + v, cuda)
    z = (3 * torch.randn(m, v + 3, generator=g, device=cuda)).to(dtype)[:, 1:v + 1]
    y = torch.randint(-1, v + 1, (m,), generator=g, device=cuda)
    y[0] = v - 1
    if m > 6:
        z[1], z[2], z[3, :v // 2], z[4] = -math.inf, torch.finfo(dtype).min, -math.inf, math.nan
        y[:6] = torch.tensor([v - 1, 0, 1, v - 1, -1, 0], device=cuda)
        z[5, 0] = -math.inf
    lp, tol, q, e, there = logp_reference(z, y)
    leaf = z.detach().clone().requires_grad_()
    out = rbg.token_logp(leaf, y)
    within(out.detach(), lp, tol)
    w = torch.randn(m, generator=g, device=cuda)
    out.backward(w)
    ref = -q * (w.double() * there)[:, None]
    ref[torch.arange(m, device=cuda), torch.where(there, y, 0)] += w.double() * there
    ref = torch.where(there[:, None], ref, 0.0)
    bound = w.double().abs()[:, None] * (q * (e + 4 * U)[:, None] + 2.0 ** -125) + stored(ref, F32) + 2 * U * w.double().abs()[:, None]
    within(leaf.grad, ref, torch.nan_to_num(bound) + stored(ref, dtype))


def packed(seed, m, pairs, dev, lead=0, behind=0):
    g = torch.Generator().manual_seed(seed)
    cuts = torch.sort(torch.randint(lead, m - behind + 1, (2 * pairs - 1,), generator=g)).values
    return torch.cat([torch.tensor([lead]), cuts, torch.tensor([m - behind])]).to(dev)


def preference_reference(lp, tol, offsets, ref, beta, smoothing):
    """(margin, its bound, loss, its bound, d loss / d margin, its bound) in 64 bits."""
    o = offsets.tolist()
    s = torch.stack([lp[a:b].sum() for a, b in zip(o[:-1], o[1:])]) - ref.double()
    t = torch.stack([tol[a:b].sum() for a, b in zip(o[:-1], o[1:])])
    h = beta * (s[0::2] - s[1::2])
    th = abs(beta) * (t[0::2] + t[1::2]) * (1 + U) + 2 * U * h.abs()
    ls = torch.nn.functional.logsigmoid
    loss = -(1 - smoothing) * ls(h) - (smoothing * ls(-h) if smoothing else 0.0)
    dh = smoothing * torch.sigmoid(h) - (1 - smoothing) * torch.sigmoid(-h)
    return h, th, loss, th + 8 * U * (loss.abs() + 1), dh, th / 4 + 8 * U  # |d loss / d h| <= 1, |d2 loss / d h2| <= 1/4


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m,v,pairs,lead,behind", [(1, 1, 1, 0, 0), (2, 3, 1, 0, 0), (40, 1683, 4, 3, 5), (256, 33, 4, 1, 0), (130, 900, 40, 0, 30), (9, 50001, 2, 0, 1), (700, 513, 300, 0, 0), (4756, 18, 2, 0, 0), (600, 9001, 5, 7, 11)])
@pytest.mark.parametrize("smoothing,beta", [(0.0, 0.1), (0.3, 1.0), (1.0, -0.5)])
def test_preference(rbg, cuda, dtype, m, v, pairs, lead, behind, smoothing, beta):
    g = gen(m + pairs, cuda)
    z = (2 * torch.randn(m, v, generator=g, device=cuda)).to(dtype)
    y = torch.randint(v, (m,), generator=g, device=cuda)
    y[torch.rand(m, generator=g, device=cuda) < 0.2] = -1
    offsets = packed(pairs, m, pairs, cuda, lead, behind)
    ref = -5 * torch.rand(2 * pairs, generator=g, device=cuda)
    weight = torch.rand(pairs, generator=g, device=cuda) + 0.5
    lp, tol, q, e, there = logp_reference(z, y)
    h, th, loss, tl, dh, td = preference_reference(lp, tol, offsets, ref, beta, smoothing)
    got, margin, grad = rbg.preference_grad(z, y, offsets, ref, beta=beta, label_smoothing=smoothing, pair_weight=weight)
    within(margin, h, th)
    within(got, loss, tl)
    c, tc = torch.zeros(m, dtype=torch.float64, device=cuda), torch.zeros(m, dtype=torch.float64, device=cuda)
    o = offsets.tolist()
    for s in range(2 * pairs):
        c[o[s]:o[s + 1]] = (1 if s % 2 == 0 else -1) * beta * dh[s // 2] * weight[s // 2].double()
        tc[o[s]:o[s + 1]] = abs(beta) * (td[s // 2] + 4 * U) * weight[s // 2].double()
    c, tc = c * there, tc * there
    want = -q * c[:, None]
    want[torch.arange(m, device=cuda), torch.where(there, y, 0)] += c
    one = torch.zeros_like(q)
    one[torch.arange(m, device=cuda), torch.where(there, y, 0)] = 1.0
    bound = tc[:, None] * (q + one) + c.abs()[:, None] * (q * (e[:, None] + 4 * U) + 2 * U) + 2.0 ** -125 + stored(want, F32)
    within(grad, want, bound + stored(want, dtype))
    assert torch.all(grad[~there] == 0) and torch.all(grad[:lead] == 0) and torch.all(grad[m - behind:] == 0)
    # the same through autograd, with a gradient for the margin too
    leaf = z.detach().clone().requires_grad_()
    l2, h2 = rbg.preference_loss(rbg.token_logp(leaf, y), offsets, ref, beta=beta, label_smoothing=smoothing)
    within(l2.detach(), loss, tl + th)
    torch.autograd.backward([l2, h2], [weight, torch.zeros_like(weight)])
    within(leaf.grad, want, 2 * bound + stored(want, dtype))
    leaf.grad = None
    rbg.preference_loss(rbg.token_logp(leaf, y), offsets, ref, beta=beta, label_smoothing=smoothing)[1].sum().backward()
    plain = torch.autograd.grad(sum((1 if s % 2 == 0 else -1) * beta * x for s, x in enumerate(_sums(leaf, y, there, o))), leaf)[0]
    within(leaf.grad, plain.double(), abs(beta) * ((e + 12 * U)[:, None] * (q + one)) + 2 * stored(plain.double(), dtype) + 2.0 ** -125)


def _sums(z, y, there, o):
    lq = torch.log_softmax(z.double(), 1)
    lp = torch.where(there, lq.gather(1, torch.where(there, y, 0)[:, None])[:, 0], 0.0)
    return [lp[a:b].sum() for a, b in zip(o[:-1], o[1:])]


def test_preference_long_sums(rbg, cuda):
    """A margin of order 1 from sums of order 1e6: 32-bit sums would lose it."""
    m = 200_000
    g = gen(1, cuda)
    logp = -5 * torch.rand(m, generator=g, device=cuda)
    offsets = torch.tensor([0, m // 2, m], device=cuda)
    sums = torch.stack([logp[:m // 2].double().sum(), logp[m // 2:].double().sum()])
    ref = sums.float() + torch.tensor([0.5, -0.25], device=cuda)
    loss, margin = rbg.preference_loss(logp, offsets, ref, beta=1.0)
    want = (sums[0] - ref[0].double()) - (sums[1] - ref[1].double())
    assert abs(float(margin[0]) - float(want)) <= 2 * U * abs(float(want)) + 1e-9
    assert abs(float(loss[0]) - math.log1p(math.exp(-float(want)))) <= 1e-6


def test_preference_extreme_margins(rbg, cuda):
    logp = torch.tensor([0.0, -2e4, -math.inf, 0.0, math.nan, 0.0, 0.0, 0.0], device=cuda)
    offsets = torch.arange(9, device=cuda)
    loss, margin = rbg.preference_loss(logp, offsets, torch.zeros(8, device=cuda), beta=1.0)
    assert float(loss[0]) == 0.0 and float(loss[1]) == math.inf and math.isnan(float(loss[2])) and abs(float(loss[3]) - math.log(2)) < 1e-6
    assert float(margin[0]) == 2e4 and float(margin[1]) == -math.inf


def test_preference_offsets_outside_are_clamped(rbg, cuda):
    logp = torch.ones(5, device=cuda)
    offsets = torch.tensor([-3, 2, 1 << 40], device=cuda)
    _, margin = rbg.preference_loss(logp, offsets, torch.zeros(2, device=cuda), beta=1.0)
    assert float(margin[0]) == 2 - 3
    z, y = torch.zeros(5, 4, device=cuda), torch.zeros(5, dtype=torch.int64, device=cuda)
    _, _, grad = rbg.preference_grad(z, y, torch.tensor([3, 1, 2], device=cuda), torch.zeros(2, device=cuda))
    assert grad.shape == (5, 4) and bool(torch.isfinite(grad).all())


def test_preference_is_bpr_for_single_tokens(rbg, cuda):
    """One token each on a shared row and no reference model: the normalizers cancel and the loss is BPR's -log sigmoid(pos - neg)."""
    g = gen(9, cuda)
    u, items = torch.randn(50, 16, generator=g, device=cuda), torch.randn(200, 16, generator=g, device=cuda)
    pos, neg = torch.randint(200, (50,), generator=g, device=cuda), torch.randint(200, (50,), generator=g, device=cuda)
    scores = rbg.score(u, items)
    y = torch.stack([pos, neg], 1).view(-1)
    loss, margin, _ = rbg.preference_grad(scores.repeat_interleave(2, 0), y, torch.arange(101, device=cuda), torch.zeros(100, device=cuda), beta=1.0)
    s = scores.double()
    want = s.gather(1, pos[:, None])[:, 0] - s.gather(1, neg[:, None])[:, 0]
    # the same row twice: the same S, and its logarithm in 64 bits cancels to the rounding of 64 bits
    within(margin, want, 2 * U * want.abs() + 1e-12)
    within(loss, -torch.nn.functional.logsigmoid(want), 8 * U * (want.abs() + 1))


# ---- 8 bits ------------------------------------------------------------------------------------------------------------

def codes_reference(x):
    """The definition: fl32(max / 127), the nearest whole number to fl32(x / scale).  (A quotient of two 32-bit numbers rounded to 64
    and then to 32 bits is the one rounded to 32 bits.)"""
    x = x.double().cpu()
    s = (x.abs().amax(1) / 127.0).float().double()
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    q = torch.where(s[:, None] > 0, (x / s[:, None]).float().double().round().clamp(-127, 127), 0.0)
    return q, s


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,k", [(1, 1), (3, 5), (33, 64), (7, 127), (5, 513), (40, 1000), (2, 8193), (1, 131071)])
def test_quantize_rows(rbg, cuda, dtype, n, k):
    g = gen(n + k, cuda)
    x = (torch.randn(n, k + 3, generator=g, device=cuda) * 10.0 ** torch.randint(-3, 4, (n, 1), generator=g, device=cuda)).to(dtype)[:, 2:k + 2]
    if n > 2:
        x[0] = 0.0
        x[1] = torch.finfo(dtype).smallest_normal / 4
        x[2] = torch.arange(k, device=cuda).to(dtype) - k // 2  # ties
    codes, scale = rbg.quantize_rows(x)
    q, s = codes_reference(x)
    assert torch.equal(codes.cpu().double(), q) and torch.equal(scale.cpu().double(), s)
    full = codes.as_strided((n, codes.stride(0)), (codes.stride(0), 1))
    assert torch.all(full[:, k:] == 0)


def test_quantize_rows_that_are_not_finite(rbg, cuda):
    x = torch.randn(4, 700, device=cuda)
    x[1, 699], x[2, 0] = math.nan, -math.inf
    codes, scale = rbg.quantize_rows(x)
    assert scale.isnan().tolist() == [False, True, True, False] and torch.all(codes[1:3] == 0)
    s = rbg.score_int8(x, *rbg.quantize_rows(torch.randn(5, 700, device=cuda)))
    assert torch.all(s[1:3].isnan()) and bool(torch.isfinite(s[::3]).all())


def scores_check(rbg, u, codes, scales, out_dtype):
    got = rbg.score_int8(u, codes, scales, out_dtype=out_dtype)
    q, s = codes_reference(u)
    ref = (q @ codes.cpu().double().t().contiguous()) * s[:, None] * scales.cpu().double()[None]  # whole-number sums below 2^53: exact
    # the sum to 32 bits, and two products
    within(got.cpu(), ref, 3.1 * U * ref.abs() + stored(ref, out_dtype) + 2.0 ** -148)
    return got


@pytest.mark.parametrize("b,n,k", [(1, 1, 1), (1, 1000, 128), (2, 333, 64), (3, 5, 7), (4, 4097, 100), (8, 130, 1000), (16, 257, 8192), (17, 129, 65), (33, 64, 4096),
                                   (130, 257, 64), (129, 130, 1000), (300, 1025, 48), (64, 300, 8208), (513, 511, 2049), (1, 3, 131071), (700, 40, 16)])
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, BF16), (F16, F32), (F32, F16)])
def test_score_int8(rbg, cuda, b, n, k, dtype, out_dtype):
    g = gen(b + n + k, cuda)
    u = torch.randn(b, k, generator=g, device=cuda).to(dtype)
    codes, scales = rbg.quantize_rows(torch.randn(n, k, generator=g, device=cuda) * 0.1)
    scores_check(rbg, u, codes, scales, out_dtype)


@pytest.mark.parametrize("b,n,k,out_dtype", [(3500, 3600, 129, F32), (4096, 4096, 1024, BF16), (2050, 8003, 300, F32), (1025, 10241, 257, F16), (256, 49153, 2048, BF16),
                                             (70, 49000, 64, F32), (1100, 40001, 250, F32), (2000, 40003, 129, BF16), (100, 1000, 2050, F32), (900, 1100, 1030, BF16), (2048, 40982, 64, F32), (333, 9001, 100, BF16), (40, 70003, 33, F16)])
def test_score_int8_many(rbg, cuda, b, n, k, out_dtype):
    """Sizes that fill the chip with large tiles or with long walks; every score against the same in 64 bits (here on the GPU), and nothing
    written outside the scores."""
    g = gen(b + k, cuda)
    u = torch.randn(b, k, generator=g, device=cuda)
    codes, scales = rbg.quantize_rows(torch.randn(n, k, generator=g, device=cuda))
    got = rbg.score_int8(u, codes, scales, out_dtype=out_dtype)
    q, s = codes_reference(u)
    ref = torch.matmul(q.to(cuda), codes.double().t().contiguous()) * s.to(cuda)[:, None] * scales.double()[None]
    within(got, ref, 3.1 * U * ref.abs() + stored(ref, out_dtype) + 2.0 ** -148)
    # rows of a wider tensor at every offset of a line: the columns beside them keep what they hold
    qu, su = torch.zeros(b, (k + 127) // 128 * 128, dtype=torch.int8, device=cuda), torch.empty(b, device=cuda)
    lib = rbg._lib.lib
    rbg._lib.check(lib.rbg_quantize_rows_i8(u.data_ptr(), k, 0, b, k, qu.data_ptr(), qu.shape[1], su.data_ptr(), torch.cuda.current_stream().cuda_stream))
    wide = torch.full((b + 1, n + 13), 77.0, dtype=out_dtype, device=cuda)
    rbg._lib.check(lib.rbg_score_i8(qu.data_ptr(), qu.shape[1], su.data_ptr(), b, codes.data_ptr(), codes.stride(0), scales.data_ptr(), n, k,
                                    wide.data_ptr() + 5 * wide.element_size(), n + 13, rbg.vocab._DTYPES[out_dtype], torch.cuda.current_stream().cuda_stream))
    assert torch.equal(wide[:b, 5:n + 5], got)
    wide[:b, 5:n + 5] = 77.0
    assert bool(torch.all(wide == 77.0))


@pytest.mark.parametrize("b,n,k", [(1, 40982, 128), (1, 77, 1), (5, 1000, 1638), (16, 300, 512), (16, 301, 513), (3, 40000, 2000)])
@pytest.mark.parametrize("dtype", ALL)
def test_score_int8_in_one_launch_or_two(rbg, cuda, b, n, k, dtype):
    """Few users' codes made where they are used, against the same codes made first: the same bits."""
    g = gen(n, cuda)
    u = torch.randn(b, k + 1, generator=g, device=cuda).to(dtype)[:, 1:]
    if b > 2:
        u[1], u[2, k // 2] = 0.0, math.inf
    codes, scales = rbg.quantize_rows(torch.randn(n, k, generator=g, device=cuda))
    qu, su = torch.zeros(b, (k + 127) // 128 * 128, dtype=torch.int8, device=cuda), torch.empty(b, device=cuda)
    st, lib = torch.cuda.current_stream().cuda_stream, rbg._lib.lib
    rbg._lib.check(lib.rbg_quantize_rows_i8(u.data_ptr(), k + 1, rbg.vocab._DTYPES[dtype], b, k, qu.data_ptr(), qu.shape[1], su.data_ptr(), st))
    want = torch.empty(b, n, device=cuda)
    rbg._lib.check(lib.rbg_score_i8(qu.data_ptr(), qu.shape[1], su.data_ptr(), b, codes.data_ptr(), codes.stride(0), scales.data_ptr(), n, k, want.data_ptr(), n, 0, st))
    got = rbg.score_int8(u, codes, scales)
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)) and torch.equal(got.isnan(), want.isnan())
    if b > 2:
        assert bool(got[2].isnan().all()) and bool((got[1] == 0).all())


def test_score_int8_exact_sums(rbg, cuda):
    """All codes at their ends: sums of 131 071 products of 127 x 127 and 127 x -128 stay whole."""
    k = 131071
    u = torch.ones(3, k, device=cuda)
    u[1] = -1.0
    codes = torch.full((130, k), 127, dtype=torch.int8, device=cuda)
    codes[5] = -128
    codes[6, 1:] = 0
    s = rbg.score_int8(u, codes, torch.ones(130, device=cuda))
    su = float(torch.tensor(1.0) / torch.tensor(127.0))
    f = lambda acc: float(torch.tensor(float(acc), dtype=F32) * torch.tensor(su, dtype=F32))  # noqa: E731
    assert float(s[0, 0]) == f(127 * 127 * k) and float(s[1, 0]) == -f(127 * 127 * k) and float(s[0, 5]) == f(-128 * 127 * k) and float(s[2, 6]) == f(127 * 127)


@pytest.mark.parametrize("b", [1, 5, 200])
@pytest.mark.parametrize("k", [7, 64, 130, 1024])
def test_score_int8_layouts(rbg, cuda, b, k):
    g = gen(k, cuda)
    u = torch.randn(b, k, generator=g, device=cuda)
    codes, scales = rbg.quantize_rows(torch.randn(150, k, generator=g, device=cuda))
    want = scores_check(rbg, u, codes, scales, F32)
    junk = torch.randint(-128, 128, (150, k + 77), generator=g, device=cuda, dtype=torch.int8)
    junk[:, 5:k + 5] = codes
    wide = torch.randint(-128, 128, (300, (k + 127) // 64 * 64), generator=g, device=cuda, dtype=torch.int8)
    wide[::2, 16:k + 16] = codes if k + 16 <= wide.shape[1] else 0
    forms = [codes.contiguous(), junk[:, 5:k + 5], codes.t().contiguous().t()] + ([wide[::2, 16:k + 16]] if k + 16 <= wide.shape[1] else [])
    for c in forms:  # (the columns behind K hold anything; rows may start anywhere)
        assert torch.equal(rbg.score_int8(u, c, scales), want)
    big = torch.randn(b, k + 5, generator=g, device=cuda)
    big[:, 2:k + 2] = u
    assert torch.equal(rbg.score_int8(big[:, 2:k + 2], codes, scales), want)
    assert rbg.score_int8(u[:0], codes, scales).shape == (0, 150) and rbg.score_int8(u, codes[:0], scales[:0]).shape == (b, 0)


def test_score_int8_beyond_32_bits(rbg, cuda):
    n = (1 << 25) + 77  # the codes' bytes pass 2^31
    codes = torch.zeros(n, 64, dtype=torch.int8, device=cuda)
    codes[-1], codes[-2, 0] = 1, 2
    s = rbg.score_int8(torch.full((1, 64), 127.0, device=cuda), codes, torch.ones(n, device=cuda))
    assert float(s[0, -1]) == 64 * 127 and float(s[0, -2]) == 2 * 127 and float(s[0, 0]) == 0
    s = rbg.score_int8(torch.full((130, 64), 127.0, device=cuda), codes[-(1 << 24):], torch.ones(1 << 24, device=cuda), out_dtype=BF16)  # 2^31 + .. scores
    assert float(s[129, -1]) == 64 * 127 and float(s[128, -2]) == 254 and float(s[129, 0]) == 0 and float(s[0, -1]) == 64 * 127


# ---- together ----------------------------------------------------------------------------------------------------------

def test_a_student_from_ids_to_table_gradient(rbg, cuda):
    """Ids -> rows -> logits -> a teacher's lists (full_sort_topk) -> loss -> gradients of the logits and of the table, all through the
    public entry points, against the same in 64 bits; then the table answers in 8 bits."""
    g = gen(21, cuda)
    n, v, d, k = 300, 1200, 32, 10
    teacher_u, teacher_i = torch.randn(n, 64, generator=g, device=cuda), torch.randn(v, 64, generator=g, device=cuda)
    val, idx = rbg.full_sort_topk(None, teacher_u, teacher_i, torch.arange(n, device=cuda), k)
    table = torch.randn(v, d, generator=g, device=cuda, requires_grad=True)
    ids = torch.randint(v, (n,), generator=g, device=cuda)
    rows = rbg.embedding(table, ids, scale=0.5, padding_idx=0)
    logits = rows @ table.t()
    loss = rbg.distill_topk(logits, idx, val, temperature=2.0)
    loss.mean().backward()
    t64 = table.detach().double().requires_grad_()
    r64 = t64[ids] * 0.5
    r64 = torch.where((ids == 0)[:, None], r64.detach(), r64)
    z64 = (r64 @ t64.t()) / 2.0
    p = torch.softmax(val.double() / 2.0, 1)
    l64 = 4.0 * (torch.xlogy(p, p) - p * torch.log_softmax(z64, 1).gather(1, idx)).sum(1)
    l64.mean().backward()
    # 32-bit products of d terms of order |row| |item| <= ~ 30: each logit is off by at most d u sum|..| < 1e-4, and d loss / d z < T
    assert float((loss.detach().double() - l64.detach()).abs().max()) < 4e-4
    assert float((table.grad.double() - t64.grad).abs().max()) < 1e-3 * float(t64.grad.abs().max())
    codes, scales = rbg.quantize_rows(table.detach())
    s8, s32 = rbg.score_int8(rows.detach(), codes, scales), rbg.score(rows.detach(), table.detach())
    # a code is off by half a step: |s8 - s| <= sum (|u| step_i / 2 + |i| step_u / 2 + ..) <= d max|u| max|i| / 127
    bound = d * rows.detach().abs().amax(1)[:, None] * table.detach().abs().amax(1)[None] / 127.0 * 1.01
    assert bool(torch.all((s8 - s32).abs() <= bound))


def all_ops(rbg, cuda, seed):
    g = gen(seed, cuda)
    table = torch.randn(500, 40, generator=g, device=cuda)
    ids = torch.randint(-1, 500, (20000,), generator=g, device=cuda)
    grad = torch.randn(20000, 40, generator=g, device=cuda)
    z, idx, val, w = distill_inputs(seed, 40, 9001, 7, BF16, cuda)
    y = torch.randint(-1, 9001, (40,), generator=g, device=cuda)
    offsets = packed(3, 40, 3, cuda)
    ref = torch.randn(6, generator=g, device=cuda)
    codes, scales = rbg.quantize_rows(torch.randn(700, 96, generator=g, device=cuda))
    u1, u2 = torch.randn(1, 96, generator=g, device=cuda), torch.randn(150, 96, generator=g, device=cuda)

    def run():
        out = [rbg.embedding(table, ids, scale=2.0), rbg.embedding_grad(grad, ids, 500), rbg.embedding_grad(grad[:3000], ids[:3000], 500)]
        out += rbg.distill_topk_grad(z, idx, val, row_weight=w)
        out += rbg.preference_grad(z, y, offsets, ref)
        out += [rbg.score_int8(u1, codes, scales), rbg.score_int8(u2, codes, scales), rbg.token_logp(z, y)]
        return out

    return run, [table, grad, z, u1, u2]


def test_captured_and_replayed(rbg, cuda):
    """Two captured graphs of every operator, replayed in turn with new inputs and eager work between the replays."""
    graphs = []
    for seed in (1, 2):
        run, inputs = all_ops(rbg, cuda, seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((run, inputs, graph, out))
    for turn in range(3):
        for run, inputs, graph, out in graphs:
            for t in inputs:
                t.mul_(-0.75)
            graph.replay()
            eager = run()
            torch.cuda.synchronize()
            for a, b in zip(out, eager):
                assert torch.equal(a, b)


def test_on_another_stream(rbg, cuda):
    run, _ = all_ops(rbg, cuda, 4)
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for out in got:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_wrappers_refuse(rbg, cuda):
    f, i = torch.zeros(2, 4, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    o3 = torch.tensor([0, 1, 2], device=cuda)
    refused = [
        (TypeError, lambda: rbg.embedding(f.double(), i)), (TypeError, lambda: rbg.embedding(f, i.float())), (ValueError, lambda: rbg.embedding(f[0], i)),
        (RuntimeError, lambda: rbg.embedding(f, i.cpu())), (ValueError, lambda: rbg.embedding_grad(f, i[:1], 3)), (TypeError, lambda: rbg.embedding_grad(f, i, 3, out_dtype=F16)),
        (ValueError, lambda: rbg.distill_topk(f, i, f[:, 0])), (ValueError, lambda: rbg.distill_topk(f, i[:, None], f)), (rbg.RbgError, lambda: rbg.distill_topk(f, i[:, None], f[:, :1], temperature=0.0)),
        (rbg.RbgError, lambda: rbg.distill_topk(f, i[:, None].expand(2, 257), f[:, :1].expand(2, 257))), (rbg.RbgError, lambda: rbg.distill_topk(f, i[:, None][:, :0], f[:, :0])),
        (ValueError, lambda: rbg.distill_topk_grad(f, i[:, None], f[:, :1], row_weight=f[0])), (rbg.RbgError, lambda: rbg.distill_topk(f[:, :0], i[:, None], f[:, :1])),
        (ValueError, lambda: rbg.token_logp(f, i[:1])), (ValueError, lambda: rbg.preference_loss(f[0], o3[:2], f[0, :1])), (ValueError, lambda: rbg.preference_loss(f[0], o3, f[0])),
        (TypeError, lambda: rbg.preference_loss(f, o3, f[0, :2])), (rbg.RbgError, lambda: rbg.preference_loss(f[0], o3, f[0, :2], label_smoothing=2.0)),
        (ValueError, lambda: rbg.preference_grad(f, i, o3, f[0, :2], pair_weight=f[0])), (ValueError, lambda: rbg.quantize_rows(f[:, :0])),
        (TypeError, lambda: rbg.score_int8(f, f, f[0])), (ValueError, lambda: rbg.score_int8(f, torch.zeros(3, 5, dtype=torch.int8, device=cuda), f[0, :3])),
        (ValueError, lambda: rbg.score_int8(f, torch.zeros(3, 4, dtype=torch.int8, device=cuda), f[0])), (TypeError, lambda: rbg.score_int8(f, torch.zeros(4, 4, dtype=torch.int8, device=cuda), f[0], out_dtype=torch.int8)),
        (rbg.RbgError, lambda: rbg.score_int8(torch.zeros(1, 131072, device=cuda), torch.zeros(1, 131072, dtype=torch.int8, device=cuda), f[0, :1])),
    ]
    for k, (error, call) in enumerate(refused):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {k} was not refused")
    for leaf in (torch.zeros(3, 4, device=cuda, requires_grad=True),):  # gradients of gradients are refused, not wrong
        (g,) = torch.autograd.grad(rbg.token_logp(leaf, torch.zeros(3, dtype=torch.int64, device=cuda)).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


@pytest.mark.parametrize("b,n", [(1, 500), (3, 33000), (16, 66000), (40, 200), (64, 2000)])
def test_scores_of_every_length(rbg, cuda, b, n):
    """Lengths that leave the waves that share a row every remainder of steps, at the sizes where 1, 2 and 4 groups of items go to a wave."""
    few = min(n, 500)
    at = torch.arange(n, device=cuda) % few
    for k in (1, 63, 64, 65, 200, 257, 1000, 1023, 1025, 1100, 1281, 1500, 1537, 1800, 2049, 2200, 2310, 2600, 3200, 4100, 4200, 5000, 8193):
        g = gen(b + k, cuda)
        u = torch.randn(b, k, generator=g, device=cuda)
        codes, scales = rbg.quantize_rows(torch.randn(few, k, generator=g, device=cuda))
        wide = torch.full((n, codes.stride(0)), 5, dtype=torch.int8, device=cuda)  # (what stands behind a row's end is read and not used)
        wide[:, :k] = codes[at]
        qu, su = rbg.quantize_rows(u)
        sums = qu.double() @ codes.double().t().contiguous()
        ref = sums.float() * su[:, None] * scales  # exact sums, then the two products in the order the operator takes them
        assert torch.equal(rbg.score_int8(u, wide[:, :k], scales[at]), ref[:, at]), (b, n, k)


# ---- more rows than one launch takes -------------------------------------------------------------------------------------

MANY = (1 << 21) + 3


def test_many_ids(rbg, cuda):
    n = (1 << 26) + 5
    table = torch.randn(97, 1, generator=gen(1, cuda), device=cuda).to(F16)
    ids = torch.arange(n, device=cuda) % 97
    out = rbg.embedding(table, ids)
    assert torch.equal(out[:, 0], table[:, 0].repeat(n // 97 + 1)[:n])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_distilled_rows(rbg, cuda, dtype):
    """The rows repeat with a period, so that every launch's rows can be held against the first ones'."""
    few = 1000
    z, idx, val, w = distill_inputs(3, few, 5, 2, dtype, cuda)
    at = torch.arange(MANY, device=cuda) % few
    loss, grad = rbg.distill_topk_grad(z[at], idx[at], val[at], row_weight=w[at])
    one, one_grad = rbg.distill_topk_grad(z, idx, val, row_weight=w)
    assert torch.equal(loss, one[at]) and torch.equal(grad, one_grad[at])
    leaf = z[at].requires_grad_()
    rbg.distill_topk(leaf, idx[at], val[at]).backward(w[at])
    few_leaf = z.clone().requires_grad_()
    rbg.distill_topk(few_leaf, idx, val).backward(w)
    assert torch.equal(leaf.grad, few_leaf.grad[at])


def test_many_pairs(rbg, cuda):
    """Pairs of one token each whose logits say which pair they belong to."""
    few = 1000
    g = gen(4, cuda)
    z, y = torch.randn(2 * few, 3, generator=g, device=cuda), torch.randint(0, 3, (2 * few,), generator=g, device=cuda)
    ref, w = torch.randn(2 * few, generator=g, device=cuda), torch.rand(few, generator=g, device=cuda)
    tok, pair = torch.arange(2 * MANY, device=cuda) % (2 * few), torch.arange(MANY, device=cuda) % few
    loss, margin, grad = rbg.preference_grad(z[tok], y[tok], torch.arange(2 * MANY + 1, device=cuda), ref[tok], beta=0.5, pair_weight=w[pair])
    l1, m1, g1 = rbg.preference_grad(z, y, torch.arange(2 * few + 1, device=cuda), ref, beta=0.5, pair_weight=w)
    assert torch.equal(loss, l1[pair]) and torch.equal(margin, m1[pair]) and torch.equal(grad, g1[tok])
    logp = rbg.token_logp(z[tok], y[tok])
    assert torch.equal(logp, rbg.token_logp(z, y)[tok])
    l2, m2 = rbg.preference_loss(logp, torch.arange(2 * MANY + 1, device=cuda), ref[tok], beta=0.5)
    l3, m3 = rbg.preference_loss(logp[:2 * few], torch.arange(2 * few + 1, device=cuda), ref, beta=0.5)
    assert torch.equal(l2, l3[pair]) and torch.equal(m2, m3[pair])


def test_many_quantized_rows(rbg, cuda):
    x = torch.randn(1000, 3, generator=gen(5, cuda), device=cuda)
    at = torch.arange(MANY, device=cuda) % 1000
    codes, scales = rbg.quantize_rows(x[at])
    c1, s1 = rbg.quantize_rows(x)
    assert torch.equal(codes, c1[at]) and torch.equal(scales, s1[at])


@pytest.mark.parametrize("b,k", [(1, 5), (2, 1100), (20, 5)])
def test_many_items(rbg, cuda, b, k):
    n = (1 << 24) + 5
    g = gen(b + k, cuda)
    u, items = torch.randn(b, k, generator=g, device=cuda), torch.randn(1000, k, generator=g, device=cuda)
    codes, scales = rbg.quantize_rows(items)
    at = torch.arange(n, device=cuda) % 1000
    wide = torch.empty(n, codes.stride(0), dtype=torch.int8, device=cuda)
    wide[:, :k] = codes[at]
    out = rbg.score_int8(u, wide[:, :k], scales[at])
    one = rbg.score_int8(u, codes, scales)  # exact sums: the same bits whatever the form
    assert all(torch.equal(out[r], one[r][at]) for r in range(b))


@pytest.mark.parametrize("n", [50, 3000])
def test_padding_row_counted_from_the_end(rbg, cuda, n):
    g = gen(n, cuda)
    grad, ids = torch.randn(n, 24, generator=g, device=cuda), torch.randint(0, 30, (n,), generator=g, device=cuda)
    got = rbg.embedding_grad(grad, ids, 30, padding_idx=-2)
    assert torch.equal(got, rbg.embedding_grad(grad, ids, 30, padding_idx=28)) and torch.all(got[28] == 0) and torch.any(got[27] != 0)
    for wrong in (30, -31):
        with pytest.raises(ValueError):
            rbg.embedding_grad(grad, ids, 30, padding_idx=wrong)
        with pytest.raises(ValueError):
            rbg.embedding(torch.zeros(30, 4, device=cuda), ids, padding_idx=wrong)


# one launch for pairs and gradients up to 1 024 tokens, 256 pairs and 32 MB of logits; three beyond
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m,v,pairs", [(1024, 33, 256), (1024, 33, 257), (1025, 33, 256), (300, 1500, 1), (1000, 4097, 3), (1024, 8192, 2), (1023, 20000, 40)])
def test_preference_forms(rbg, cuda, dtype, m, v, pairs):
    """A log-probability is off by its row's S and its own z - m in 32 bits; a margin by those of its tokens, summed in 64 bits, and its own
    rounding; the sigmoid passes a margin's error on by at most a quarter of it."""
    g = gen(m + pairs, cuda)
    z = torch.randn(m, v, generator=g, device=cuda).to(dtype)
    y = torch.randint(-1, v, (m,), generator=g, device=cuda)
    offsets = torch.sort(torch.randint(0, m + 1, (2 * pairs + 1,), generator=g, device=cuda)).values
    weight = torch.rand(pairs, generator=g, device=cuda) + 0.5
    lp = torch.log_softmax(z.double(), 1)
    lp = torch.where(y >= 0, lp.gather(1, y.clamp(min=0)[:, None])[:, 0], 0.0)
    sums = torch.cat([lp.new_zeros(1), lp.cumsum(0)])[offsets]
    seq = sums[1:] - sums[:-1]
    ref = (seq + torch.randn(2 * pairs, generator=g, device=cuda)).float()
    beta = 0.5
    loss, margin, grad = rbg.preference_grad(z, y, offsets, ref, beta=beta, pair_weight=weight)
    want = beta * ((seq[0::2] - ref[0::2].double()) - (seq[1::2] - ref[1::2].double()))
    # a log-probability in the call: its row's S and its own z - m in 32 bits, as in the head of this file
    spread = (z.double().amax(1) - z.double().amin(1)).max().item() / math.log(2)
    one = (4 + 3 * spread + 2 * (v / 64 + 96)) * U
    count = (offsets[1:] - offsets[:-1]).double()
    tol = beta * (count[0::2] + count[1::2]) * one + 4 * U * want.abs() + 1e-12 * seq.abs().max()
    within(margin, want, tol)
    dl = -torch.sigmoid(-want)
    where = torch.bucketize(torch.arange(m, device=cuda), offsets, right=True) - 1
    inside = (where >= 0) & (where < 2 * pairs) & (y >= 0)
    pair = where.clamp(0, 2 * pairs - 1) // 2
    w = torch.where(inside, beta * (dl * weight.double())[pair] * (1 - 2 * (where % 2)), 0.0)
    q = torch.softmax(z.double(), 1)
    hot = torch.zeros_like(q)
    hot[torch.arange(m, device=cuda)[y >= 0], y[y >= 0]] = 1.0
    want_grad = w[:, None] * (hot - q)
    # w: the sigmoid's 8 u and a quarter of the margin's error; q: its error; the difference and the product one u each
    bound = want_grad.abs() * (12 * U) + beta * weight.max() * (tol[pair] / 4)[:, None] * inside[:, None] * (hot + q) + w.abs()[:, None] * q * one
    within(grad, want_grad, bound + stored(want_grad, dtype) + stored(bound, dtype))
    assert torch.all(grad[~inside] == 0)


@pytest.mark.parametrize("n,rows,d", [(12288, 40, 24), (12289, 40, 24), (13000, 17, 9), (13000, 260000, 8), (20000, 3, 8), (40000, 200, 33), (60000, 3001, 8), (65536, 9, 4),
                                      (70000, 1000, 16), (300000, 33, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_grad_rows_between_long_runs(rbg, cuda, dtype, n, rows, d):
    """Only every third row is used and the last used one has half of the places: what lies between long runs is zeroed."""
    g = gen(n + rows, cuda)
    grad = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    ids = torch.randint(0, (rows + 2) // 3, (n,), generator=g, device=cuda) * 3
    ids[torch.rand(n, generator=g, device=cuda) < 0.5] = (rows - 1) // 3 * 3
    got = rbg.embedding_grad(grad, ids, rows)
    ref, mag, cnt = runs_reference(grad, ids, rows, 1.0, -1)
    within(got, ref, stored(ref, dtype) + mag * U * (cnt + 4))  # cnt additions in some order
    assert torch.all(got[cnt[:, 0] == 0] == 0)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("b,n", [(17, 40), (33, 1000), (100, 3000), (300, 9001), (2097153, 2)])
def test_scores_of_short_rows(rbg, cuda, dtype, b, n):
    """Users' rows of up to 128 values, whose codes the product makes on the way: those of quantize_rows, to the bit; a zero row scores
    zero, one that is not finite scores NaN."""
    for k in (1, 15, 16, 17, 32, 33, 63, 64, 65, 100, 127, 128, 129) if b < 1000 else (5,):
        g = gen(b + k, cuda)
        u = torch.randn(b, k + 3, generator=g, device=cuda).to(dtype)[:, :k]
        u[1] = 0
        u[2, k - 1], u[b - 1, 0] = math.inf, math.nan
        codes, scales = rbg.quantize_rows(torch.randn(n, k, generator=g, device=cuda))
        qu, su = rbg.quantize_rows(u)
        sums = qu.double() @ codes.double().t().contiguous()
        ref = sums.float() * su[:, None] * scales  # exact sums, then the two products in the order the operator takes them
        assert torch.isnan(ref[2]).all() and torch.isnan(ref[b - 1]).all() and (ref[1] == 0).all()
        got = rbg.score_int8(u, codes, scales)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got.nan_to_num(), ref.nan_to_num()), k


def test_a_last_slice_of_few_long_rows(rbg, cuda):
    """2^21 + 3 rows of 8 192 logits: the three rows that a launch of their own takes are not split as three rows alone would be (the call has
    no workspace for that), and come out as the same rows in a call of 1 000."""
    few, v = 1000, 8192
    z, idx, val, w = distill_inputs(5, few, v, 4, BF16, cuda)
    y = torch.randint(-1, v, (few,), generator=gen(6, cuda), device=cuda)
    at = torch.arange(MANY, device=cuda) % few
    many = z[at]  # 34 GB
    logp = rbg.token_logp(many, y[at])
    assert torch.equal(logp, rbg.token_logp(z, y)[at])
    one, one_grad = rbg.distill_topk_grad(z, idx, val, row_weight=w)
    assert torch.equal(rbg.distill_topk(many, idx[at], val[at]), one[at])
    loss, grad = rbg.distill_topk_grad(many, idx[at], val[at], row_weight=w[at])
    assert torch.equal(loss, one[at]) and torch.equal(grad[-5 * few:], one_grad[at[-5 * few:]]) and torch.equal(grad[:few], one_grad)
    del grad
    # pairs of whole blocks of `few` tokens but for the last, which holds what is left
    cuts = torch.cat([torch.arange(0, MANY, few, device=cuda)[:2 * (MANY // (2 * few))], torch.tensor([MANY], device=cuda)])
    sums = torch.stack([part.double().sum() for part in logp.split((cuts[1:] - cuts[:-1]).tolist())])
    loss, margin, grad = rbg.preference_grad(many, y[at], cuts, sums.float(), beta=0.5)
    want = 0.5 * ((sums[0::2] - sums[0::2].float().double()) - (sums[1::2] - sums[1::2].float().double()))
    # logp is rounded to 32 bits out of the call and not in it: half a step of each, in up to 2 few + few tokens of a pair
    step = (2 * U) * logp.abs().max().double()
    within(margin, want, 0.5 * 3.2 * few * step / 2 + 2 * U * want.abs())
    assert grad.shape == many.shape and bool(torch.isfinite(grad[-few:]).all()) and torch.all(grad[-few:][y[at[-few:]] < 0] == 0)


@pytest.mark.parametrize("smoothing", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("pairs,each", [(4, 1), (32, 4), (100, 5), (300, 2)])
def test_preference_is_rounded_once(rbg, cuda, smoothing, pairs, each):
    """Rows of two equal logits: a token's log-probability is -log 2 in 64 bits, its softmax 1/2 exactly, and its gradient half the pair's
    coefficient.  Margin, loss and coefficient then show their own rounding alone, half a step (and what 64 bits lose, below 2^-40):
    in the one launch of few tokens, in the pairs that the rows' workgroups form, and in the pairs' own launch."""
    g = gen(pairs, cuda)
    m = 2 * pairs * each
    beta, e = 0.75, float(torch.tensor(smoothing, dtype=F32))  # (the operator takes 32 bits)
    h = torch.linspace(-30, 30, pairs, device=cuda)
    ref = torch.stack([-h / beta, torch.rand(pairs, generator=g, device=cuda)], 1).view(-1)
    weight = torch.rand(pairs, generator=g, device=cuda) + 0.5
    h = beta * (ref[1::2].double() - ref[0::2].double())  # (both sequences of a pair sum to the same)
    offsets = torch.arange(2 * pairs + 1, device=cuda) * each
    y = torch.zeros(m, dtype=torch.int64, device=cuda)
    want = (1 - e) * (-h).clamp(min=0) + e * h.clamp(min=0) + torch.exp(-h.abs()).log1p()
    d = e * torch.sigmoid(h) - (1 - e) * torch.sigmoid(-h)
    once = U + 2.0 ** -40
    loss, margin, grad = rbg.preference_grad(torch.zeros(m, 2, device=cuda), y, offsets, ref, beta=beta, label_smoothing=smoothing, pair_weight=weight)
    within(margin, h, once * h.abs())
    within(loss, want, once * want)
    coef = (beta * d * weight.double())[:, None, None] * torch.tensor([1.0, -1.0], device=cuda)[None, :, None]
    half = coef.expand(pairs, 2, each).reshape(m) / 2
    # e sigma(h) - (1 - e) sigma(-h) cancels near a margin of log((1 - e) / e): off by 64 bits' rounding of its terms
    tol = once * half.abs() + 2.0 ** -48
    within(grad[:, 0], half, tol)
    within(grad[:, 1], -half, tol)
    # from given log-probabilities; backward from the margin that came out
    logp = torch.zeros(m, device=cuda, requires_grad=True)
    loss, margin = rbg.preference_loss(logp, offsets, ref, beta=beta, label_smoothing=smoothing)
    within(margin.detach(), h, once * h.abs())
    within(loss.detach(), want, once * want)
    loss.backward(weight)
    h = margin.detach().double()
    d = e * torch.sigmoid(h) - (1 - e) * torch.sigmoid(-h)
    coef = (beta * d * weight.double())[:, None, None] * torch.tensor([1.0, -1.0], device=cuda)[None, :, None]
    within(logp.grad, coef.expand(pairs, 2, each).reshape(m), once * coef.abs().expand(pairs, 2, each).reshape(m) + 2.0 ** -47)


def test_forward_mode_is_refused(rbg, cuda):
    """A tangent is refused by every differentiable operator, never dropped; values inside a forward-mode level are what they are outside."""
    from torch.autograd import forward_ad
    g = gen(3, cuda)
    t, dt = torch.randn(6, 8, generator=g, device=cuda), torch.randn(6, 8, generator=g, device=cuda)
    ids, offsets, ref = torch.arange(6, device=cuda), torch.tensor([0, 3, 6], device=cuda), torch.zeros(2, device=cuda)
    calls = [lambda x: rbg.embedding(x, ids, scale=2.0), lambda x: rbg.distill_topk(x, ids[:, None], t[:, :1]), lambda x: rbg.token_logp(x, ids),
             lambda x: rbg.preference_loss(x[:, 0].contiguous(), offsets, ref)[0]]
    want = [call(t) for call in calls]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, dt)
        for call, value in zip(calls, want):
            assert torch.equal(call(t), value)
            for grad_mode in (True, False):
                with torch.set_grad_enabled(grad_mode), pytest.raises((RuntimeError, NotImplementedError)):
                    call(dual)
    assert all(torch.equal(call(t), value) for call, value in zip(calls, want))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("d", [3, 64, 520])
def test_embedding_of_no_row_is_zero_at_any_scale(rbg, cuda, dtype, d):
    """1e39 and more are infinite in the operator's 32 bits: rows are scaled to infinities, places without a row stay zero."""
    ids = torch.tensor([0, -1, 4, 5, 1 << 40, 2], device=cuda)
    there = torch.tensor([True, False, True, False, False, True], device=cuda)
    for scale in (1e39, -math.inf, math.nan, -1.0):
        out = rbg.embedding(torch.ones(5, d, dtype=dtype, device=cuda), ids, scale=scale)
        assert torch.all(out[~there] == 0)
        assert bool(out[there].isnan().all()) if math.isnan(scale) else torch.all(out[there] == scale)


@pytest.mark.parametrize("b,n,k", [(1, 100, 128), (2, 333, 1100), (16, 40000, 2100), (40, 300, 64), (200, 3000, 100), (100, 500, 128), (33, 300, 300), (300, 300, 8192), (600, 1000, 300),
                                   (3000, 4200, 200), (4096, 4096, 260)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_of_large_users_and_small_items(rbg, cuda, dtype, b, n, k):
    """Scores that 32 bits hold although a user's scale times the sum passes them (1e36 / 127 times up to 127 x 127 x K): finite in every form."""
    g = gen(b + n, cuda)
    u = torch.randn(b, k, generator=g, device=cuda)
    u[::3] *= 1e36 / u[::3].abs().amax(1, keepdim=True)
    u[1::3] *= 1e-30
    u = u.to(dtype)
    codes, scales = rbg.quantize_rows(torch.randn(n, k, generator=g, device=cuda) * 10.0 ** torch.randint(-30, -5, (n, 1), generator=g, device=cuda))
    q, s = codes_reference(u)
    sums = torch.matmul(q.to(cuda), codes.double().t().contiguous())
    ref = sums * s.to(cuda)[:, None] * scales.double()[None]
    assert float((sums * s.to(cuda)[:, None]).abs().max()) > torch.finfo(F32).max > float(ref.abs().max()) * 100
    within(rbg.score_int8(u, codes, scales), ref, 3.1 * U * ref.abs() + stored(ref, F32) + 2.0 ** -148)


def test_columns_whose_bytes_pass_31_bits(rbg, cuda):
    d = (1 << 29) + 3
    table = (torch.arange(d, device=cuda) % 251).float()[None].repeat(2, 1)
    out = rbg.embedding(table, torch.tensor([1, -1], device=cuda), scale=2.0)
    assert torch.equal(out[0], 2 * table[1]) and torch.all(out[1] == 0)


def test_columns_beyond_32_bits_are_refused(rbg, cuda):
    """Widths whose lower 32 bits are a small size are not taken for it."""
    wide = torch.empty(1, (1 << 32) + 8, dtype=BF16, device=cuda)
    ids = torch.zeros(1, dtype=torch.int64, device=cuda)
    for call in (lambda: rbg.embedding(wide, ids), lambda: rbg.embedding_grad(wide, ids, 2)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,v", [(40, 50), (600, 700), (1500, 64)])
@pytest.mark.parametrize("where", ["ends", "all before", "all behind"])
def test_preference_offsets_outside_in_every_form(rbg, cuda, dtype, m, v, where):
    """Ascending offsets that begin below 0 and end behind the last token are those offsets clamped, in the one launch of few tokens, in the
    two of up to 1 024 and in the three beyond; every element of the gradient is written.  Bounds as in test_preference."""
    g = gen(m, cuda)
    z, y = torch.randn(m, v, generator=g, device=cuda).to(dtype), torch.randint(-1, v, (m,), generator=g, device=cuda)
    offsets = {"ends": [-7, m // 5, m // 5, m // 2, m - 3, m + 1, m + 50], "all before": [-(1 << 40), -9, -4, -4, -1, 0, m // 3],
               "all behind": [m // 3, m, m + 1, m + 1, m + 2, m + 9, 1 << 40]}[where]
    pairs, beta = 3, 0.5
    offsets = torch.tensor(offsets, device=cuda)
    ref = torch.randn(2 * pairs, generator=g, device=cuda)
    lp, tol, q, e, there = logp_reference(z, y)
    o = offsets.clamp(0, m)
    h, th, want_loss, tl, dh, td = preference_reference(lp, tol, o, ref, beta, 0.0)
    c, tc = torch.zeros(m, dtype=torch.float64, device=cuda), torch.zeros(m, dtype=torch.float64, device=cuda)
    for s in range(2 * pairs):
        at = slice(int(o[s]), int(o[s + 1]))
        c[at], tc[at] = (1 if s % 2 == 0 else -1) * beta * dh[s // 2], beta * (td[s // 2] + 4 * U)
    c, tc = c * there, tc * there
    one = torch.zeros_like(q)
    one[torch.arange(m, device=cuda), torch.where(there, y, 0)] = 1.0
    want = c[:, None] * (one - q)
    bound = tc[:, None] * (q + one) + c.abs()[:, None] * (q * (e[:, None] + 4 * U) + 2 * U) + 2.0 ** -125 + stored(want, F32) + stored(want, dtype)
    lib, b = rbg._lib.lib, ctypes.c_int64()
    rbg._lib.check(lib.rbg_preference_grad_workspace(m, v, ctypes.byref(b)))
    work = torch.empty(b.value, dtype=torch.uint8, device=cuda)
    loss, margin, grad = torch.full((pairs,), 77.0, device=cuda), torch.full((pairs,), 77.0, device=cuda), torch.full((m, v + 3), 77.0, dtype=dtype, device=cuda)
    rbg._lib.check(lib.rbg_preference_grad(z.data_ptr(), v, rbg.vocab._DTYPES[dtype], m, v, y.data_ptr(), offsets.data_ptr(), pairs, ref.data_ptr(), beta, 0.0, None,
                                           loss.data_ptr(), margin.data_ptr(), grad.data_ptr(), v + 3, work.data_ptr(), torch.cuda.current_stream().cuda_stream))
    within(margin, h, th)
    within(loss, want_loss, tl)
    within(grad[:, :v], want, bound)
    assert torch.all(grad[:, v:] == 77.0)
    logp = lp.float().requires_grad_()
    got, _ = rbg.preference_loss(logp, offsets, ref, beta=beta)
    within(got.detach(), want_loss, tl + beta * m * U * lp.abs().max())
    got.sum().backward()
    within(logp.grad, torch.where(there, c, logp.grad.double()), tc + beta * beta * m * U * lp.abs().max() + 2 * U * c.abs())


def test_captured_forward_and_backward(rbg, cuda):
    """A training step's forward and backward of every differentiable operator in one captured graph, replayed with new inputs and eager work
    between the replays."""
    g = gen(31, cuda)
    n, v, d, k = 700, 1500, 24, 8
    table = torch.randn(v, d, generator=g, device=cuda)
    ids, y = torch.randint(-1, v, (n,), generator=g, device=cuda), torch.randint(-1, v, (n,), generator=g, device=cuda)
    idx, val = torch.randint(-1, v, (n, k), generator=g, device=cuda), torch.randn(n, k, generator=g, device=cuda)
    offsets, ref = packed(5, n, 6, cuda, 3, 4), torch.randn(12, generator=g, device=cuda)

    def step():
        leaf = table.detach().requires_grad_()
        logits = rbg.embedding(leaf, ids, scale=0.5, padding_idx=3) @ table.t()
        z = logits.detach().requires_grad_()
        loss, margin = rbg.preference_loss(rbg.token_logp(z, y), offsets, ref)
        total = rbg.distill_topk(z, idx, val, temperature=2.0).sum() + loss.sum() + margin.sum()
        (dz,) = torch.autograd.grad(total, z)
        (dt,) = torch.autograd.grad(logits, leaf, dz)
        return total.detach(), dz, dt

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        table.mul_(-0.9)
        val.add_(0.1)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        # (the sum of the losses is torch's own: its order may differ by capture)
        assert abs(float(out[0]) - float(eager[0])) <= 1e-4 * abs(float(eager[0])) and torch.equal(out[1], eager[1]) and torch.equal(out[2], eager[2])


def test_nothing_to_do_through_autograd(rbg, cuda):
    """Calls of no rows, no pairs or no tokens have outputs and gradients of those shapes."""
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    for z in (torch.zeros(0, 5, device=cuda, requires_grad=True),):
        (rbg.distill_topk(z, none[:, None].expand(0, 3), torch.zeros(0, 3, device=cuda)).sum() + rbg.token_logp(z, none).sum()).backward()
        assert z.grad.shape == (0, 5)
    table = torch.ones(4, 3, device=cuda, requires_grad=True)
    rbg.embedding(table, none).sum().backward()
    assert torch.all(table.grad == 0)
    one = torch.zeros(1, dtype=torch.int64, device=cuda)
    for m in (0, 3, 300, 1100):
        z, y = torch.randn(m, 7, device=cuda), torch.zeros(m, dtype=torch.int64, device=cuda)
        loss, margin, grad = rbg.preference_grad(z, y, one, torch.zeros(0, device=cuda))  # no pairs
        assert loss.shape == margin.shape == (0,) and grad.shape == (m, 7) and torch.all(grad == 0)
        logp = torch.zeros(m, device=cuda, requires_grad=True)
        rbg.preference_loss(logp, one, torch.zeros(0, device=cuda))[0].sum().backward()
        assert torch.all(logp.grad == 0)
        loss, margin, grad = rbg.preference_grad(z, y, one.expand(5), torch.zeros(4, device=cuda))  # pairs of no tokens
        assert torch.all(margin == 0) and bool(torch.allclose(loss, torch.full_like(loss, math.log(2)))) and torch.all(grad == 0)
