"""The training operators (mpemu.functional) against plain implementations in 64 bits.

Tolerances.  A stored value is off by at most half a step of its type, eps(t) / 2 relative to it (fp16: 2^-25 absolute below
its normal range).  A sum of n terms in fp32 is off by at most n steps of 2^-24 (additions rounded to nearest) or 2^-23 (the
matrix unit may cut) of the sum of the terms' magnitudes.  Norms are summed in 64 bits and rounded to fp32 once."""
import math

import pytest
import torch

from mpemu import functional as F
from mpemu.cmodel import simple
from mpemu.pytquant.hip import _binding as hip

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIXTEEN = TYPES[1:]
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


@pytest.fixture(params=["native", "ctypes"])
def front(request, monkeypatch):
    """Both ways to the kernels: the C++ front and the ctypes binding."""
    if request.param == "ctypes":
        monkeypatch.setattr(F, "_native", lambda: None)
    else:
        assert F._native() is not None
    return request.param


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=gen(seed), device=DEV) * std).to(dtype)


def close(got, want, slack, what=""):
    """|got - want| <= slack + half a step of got's type."""
    bound = slack + want.abs() * (torch.finfo(got.dtype).eps / 2) + TINY[got.dtype]
    d = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((d <= bound).all()), "%s: off by %g over the bound at %s" % (
        what, float((d - bound).max()), (d - bound).argmax().item())


# ---- rows by group ------------------------------------------------------------------------------------------------------
def check_group(ids, groups):
    order, offsets = F.group_rows(ids, groups)
    flat = ids.reshape(-1).cpu().long()
    key = torch.where((flat >= 0) & (flat < groups), flat, groups)
    want = torch.sort(key, stable=True).indices
    assert order.dtype == offsets.dtype == torch.int32 and tuple(offsets.shape) == (groups + 1,)
    assert torch.equal(order.cpu().long(), want)
    assert torch.equal(offsets.cpu().long(), torch.searchsorted(key[want], torch.arange(groups + 1)))


@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 511, 4095, 4096, 4097, 20000, 4096 * 32 + 1, 4096 * 70 + 5])
@pytest.mark.parametrize("groups", [1, 2, 8, 1023, 1024, 30522])
def test_group_rows(n, groups):
    ids = torch.randint(0, groups, (n,), generator=gen(n + groups), device=DEV)
    check_group(ids, groups)


@pytest.mark.parametrize("groups", [(1 << 20) - 1, 1 << 20, (1 << 22) + 3])
@pytest.mark.parametrize("n", [1, 3000, 9000])
def test_group_rows_many_groups(n, groups):
    """One digit more than two passes hold, and the sizes around it."""
    check_group(torch.randint(0, groups, (n,), generator=gen(n), device=DEV), groups)


def test_group_rows_outside_int32_and_shapes(front):
    ids = torch.tensor([[3, -1, 0, 9], [2 ** 40, 3, -2 ** 63, 0]], device=DEV)
    check_group(ids, 4)
    check_group(ids.clamp(-5, 100).int(), 4)
    check_group(ids.t(), 4)                                  # not contiguous
    check_group(torch.full((5000,), 7, device=DEV), 3)       # nobody has a group
    check_group(torch.full((9000,), 1, device=DEV, dtype=torch.int32)[::3], 3)


# ---- embedding ----------------------------------------------------------------------------------------------------------
def embedding_reference(ids, weight, scale, padding, dout):
    flat, wide = ids.reshape(-1), weight.double()
    known = (flat >= 0) & (flat < weight.shape[0])
    out = wide[flat.clamp(0, weight.shape[0] - 1)] * scale
    out[~known] = math.nan
    counted = known if padding is None else known & (flat != padding % weight.shape[0])
    d = dout.double().reshape(-1, weight.shape[1])[counted] * scale
    dweight = torch.zeros_like(wide).index_add_(0, flat[counted], d)
    size = torch.zeros_like(wide).index_add_(0, flat[counted], d.abs())
    count = torch.bincount(flat[counted], minlength=weight.shape[0]).double()
    return out.reshape(tuple(ids.shape) + (weight.shape[1],)), dweight, size * (count + 2).unsqueeze(1) * 2.0 ** -24


def check_embedding(ids, weight, scale, padding, seed=5):
    weight = weight.detach().requires_grad_(True)
    out = F.embedding(ids, weight, scale=scale, padding_idx=padding)
    dout = randn(out.shape, out.dtype, seed)
    dweight, = torch.autograd.grad(out, (weight,), dout)
    want, dwant, slack = embedding_reference(ids, weight.detach(), scale, padding, dout)
    nan = want.isnan()
    assert torch.equal(out.isnan(), nan) and out.dtype == weight.dtype
    close(out.detach()[~nan], want[~nan], want[~nan].abs() * 2.0 ** -24, "out")
    close(dweight, dwant, slack, "dweight")
    with torch.no_grad():
        assert torch.equal(F.embedding(ids, weight, scale=scale)[~nan], out.detach()[~nan])
    return dweight


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,vocab,width", [(1, 30522, 768), (7, 1, 5), (64, 100, 64), (1023, 50, 33), (5000, 1000, 130),
                                                (300, 70000, 8), (2048, 512, 1), (100, 300, 4100)])
def test_embedding(dtype, tokens, vocab, width):
    ids = torch.randint(0, vocab, (tokens,), generator=gen(tokens), device=DEV)
    check_embedding(ids, randn((vocab, width), dtype, 1), 27.75, None)


@pytest.mark.parametrize("dtype,vocab,width", [(torch.float16, 100003, 1030), (torch.float32, 50001, 1027), (torch.bfloat16, 101, 1025)])
def test_embedding_larger_than_the_cache(dtype, vocab, width):
    """Table and rows of more than 192 MB: cleared and read past the caches; rows that begin at any element."""
    tokens = 100001 if vocab < 1000 else 3001
    ids = (torch.rand(tokens, generator=gen(7), device=DEV) ** 3 * vocab).long()   # the first entries often
    check_embedding(ids, randn((vocab, width), dtype, 1), 0.75, vocab - 1)


@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_frequent_entries(dtype):
    """Runs that fill chunks, end inside one, begin inside one, and one entry with nearly everything."""
    ids = torch.cat([torch.full((31,), 3), torch.full((33,), 4), torch.full((640,), 9), torch.full((32,), 11),
                     torch.full((9000,), 40), torch.arange(0, 60)])
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(3))].to(DEV)
    check_embedding(ids, randn((64, 200), dtype, 2), 1.0, None)
    check_embedding(torch.full((70000,), 2, device=DEV), randn((5, 24), dtype, 2), 0.5, None)


def test_embedding_padding_outside_shapes(front):
    ids = torch.tensor([[0, 5, 5, 0], [-1, 9, 10, 2 ** 40], [1, 1, 1, 0]], device=DEV)
    w = randn((10, 12), torch.float32, 3)
    dweight = check_embedding(ids, w, 2.0, 0)
    assert float(dweight[0].abs().sum()) == 0.0 and float(dweight[1].abs().sum()) > 0.0
    check_embedding(ids.clamp(-1, 10).int(), w.half(), 2.0, -1)          # the last entry pads
    check_embedding(ids.t(), w.bfloat16(), 1.5, None)                      # ids not contiguous
    check_embedding(ids, randn((12, 10), torch.float32, 4).t(), 1.0, None)   # weight not contiguous
    check_embedding(torch.zeros(0, 3, dtype=torch.int64, device=DEV), w, 1.0, None)
    check_embedding(torch.tensor(4, device=DEV), w, 1.0, None)             # 0-d


def test_embedding_views_at_odd_addresses():
    for dtype in TYPES:
        flat = randn((1 + 50 * 16,), dtype, 6)
        check_embedding(torch.randint(0, 50, (90,), generator=gen(1), device=DEV), flat[1:].view(50, 16), 3.0, None)


def test_embedding_broadcast_gradient(front):
    """A sum's gradient is one number seen through strides of zero."""
    w = randn((20, 16), torch.float32, 7).requires_grad_(True)
    ids = torch.tensor([1, 1, 2, 19], device=DEV)
    F.embedding(ids, w, scale=0.5).sum().backward()
    want = torch.zeros(20, 16, device=DEV)
    want[1], want[2], want[19] = 1.0, 0.5, 0.5
    assert torch.equal(w.grad, want)


def test_embedding_gradient_against_differences():
    w = randn((6, 4), torch.float32, 8)
    ids, v = torch.tensor([0, 3, 3, 5], device=DEV), randn((4, 4), torch.float32, 9)

    def f(t):
        return float((F.embedding(ids, t, scale=1.25).double() * v.double()).sum())

    g, = torch.autograd.grad((F.embedding(ids, w.requires_grad_(True), scale=1.25) * v).sum(), (w,))
    w = w.detach()
    for i, j in ((0, 0), (3, 2), (5, 3), (1, 1)):
        d = torch.zeros_like(w)
        d[i, j] = 0.5    # linear: any step will do; fp32 products of about 1 are off by 2^-24 each
        assert abs((f(w + d) - f(w - d)) - float(g[i, j])) < 32 * 2.0 ** -22


def test_embedding_refusals(front):
    w, ids = randn((10, 4), torch.float32, 1), torch.tensor([1], device=DEV)
    for bad in (lambda: F.embedding(ids, w[0]), lambda: F.embedding(ids, w, padding_idx=10), lambda: F.embedding(ids, w, padding_idx=-11),
                lambda: F.embedding(ids, w[:0])):
        with pytest.raises(ValueError):
            bad()
    out = F.embedding(ids, w.requires_grad_(True))
    with pytest.raises(RuntimeError):   # once only: no silent zero for the second derivative
        g, = torch.autograd.grad(out.sum(), (w,), create_graph=True)
        torch.autograd.grad(g.sum(), (w,))


@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_forward_mode_derivatives_are_refused(front, leaf, grad_mode):
    """No result without its tangent: of the calls, and of the gradients when only the incoming one carries it."""
    from torch.autograd import forward_ad
    table, x, w = randn((10, 8), torch.float32, 1), randn((6, 8), torch.float32, 2), randn((2, 8, 4), torch.float32, 3)
    ids, o = torch.tensor([1, 3, 9], device=DEV), torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV)
    y, h = F.grouped_mm(x.clone().requires_grad_(True), w.clone().requires_grad_(True), o), F.embedding(ids, table.clone().requires_grad_(True))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        def dual(t):
            return forward_ad.make_dual(t.clone().requires_grad_(leaf), torch.ones_like(t))
        for call in (lambda: F.embedding(ids, dual(table)), lambda: F.grouped_mm(dual(x), w, o), lambda: F.grouped_mm(x, dual(w), o),
                     lambda: F.grouped_mm(x, dual(w.transpose(1, 2).contiguous()).transpose(1, 2), o),
                     lambda: y.backward(dual(y.detach()), retain_graph=True), lambda: h.backward(dual(h.detach()), retain_graph=True),
                     lambda: F.grad_norm([dual(x)]), lambda: F.clip_grads_([x.clone(), dual(x)], 1.0),
                     lambda: F.clip_grads_([x], 1.0, out=[dual(x)])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    y.sum().backward()    # and everything else goes on
    h.sum().backward()


# ---- products by group --------------------------------------------------------------------------------------------------------
def offsets_of(sizes, first=0, dtype=torch.int32):
    return torch.tensor([first] + [first + sum(sizes[:i + 1]) for i in range(len(sizes))], dtype=dtype, device=DEV)


def check_grouped(x, weight, offsets, seed=11):
    """y and both gradients; dy is random.  Rows of no group get zeros whatever x holds there."""
    x, weight = x.detach().requires_grad_(True), weight.detach().requires_grad_(True)
    y = F.grouped_mm(x, weight, offsets)
    dy = randn(y.shape, y.dtype, seed)
    dx, dw = torch.autograd.grad(y, (x, weight), dy)
    X, W, DY, o = x.detach().double(), weight.detach().double(), dy.double(), offsets.tolist()
    want = [torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (y, x, weight)]
    slack = [torch.zeros_like(t) for t in want]
    u = 2.0 ** -24 if x.dtype == torch.float32 else 2.0 ** -23
    for g in range(weight.shape[0]):
        r = slice(o[g], o[g + 1])
        for k, (a, b, at) in enumerate(((X[r], W[g], r), (DY[r], W[g].t(), r), (X[r].t(), DY[r], g))):
            want[k][at] = a @ b
            slack[k][at] = (a.abs() @ b.abs()) * ((a.shape[1] + 1) * u)
    for got, w, s, what in zip((y.detach(), dx, dw), want, slack, ("y", "dx", "dweight")):
        assert got.dtype == x.dtype
        close(got, w, s, what)
    with torch.no_grad():
        assert torch.equal(F.grouped_mm(x, weight, offsets), y.detach())
    return y.detach(), dx, dw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("linear", [False, True])
@pytest.mark.parametrize("sizes,K,N", [([1], 64, 64), ([1, 0, 2, 0], 128, 96), ([130, 1, 255, 0, 64], 200, 264), ([5, 300], 33, 65),
                                       ([257, 128, 129], 64, 520), ([16] * 70, 256, 48), ([3, 1], 1, 1), ([0, 0], 40, 24),
                                       ([700, 0, 5], 1032, 136)])
def test_grouped_mm(dtype, linear, sizes, K, N):
    M, G = sum(sizes), len(sizes)
    x = randn((M, K), dtype, 1)
    w = randn((G, N, K), dtype, 2).transpose(1, 2) if linear else randn((G, K, N), dtype, 2)
    check_grouped(x, w, offsets_of(sizes))


RAGGED = [900, 0, 333, 129, 127, 600, 8, 3]


@pytest.mark.parametrize("linear", [False, True])
@pytest.mark.parametrize("dtype,sizes,K,N", [(t, RAGGED, 72, 2056) for t in TYPES]             # tiles of 128 x 128, in whole
                         + [(t, RAGGED, 77, 4109) for t in TYPES]                              # vectors or not,
                         + [(t, [1500, 300, 257, 0, 1200, 600, 1000, 100], 2056, 8264) for t in TYPES[1:]])   # and of 256 x 256
def test_grouped_mm_large(dtype, linear, sizes, K, N):
    M, G = sum(sizes), len(sizes)
    x = randn((M + 300, K), dtype, 1)
    x[M:] = math.nan
    w = randn((G, N, K), dtype, 2).transpose(1, 2) if linear else randn((G, K, N), dtype, 2)
    y, dx, dw = check_grouped(x, w, offsets_of(sizes))
    assert float(y[M:].abs().sum()) == 0.0 and float(dx[M:].abs().sum()) == 0.0


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("sizes,K,N", [([2, 0, 5, 1] * 8, 1032, 1160),      # a weight gradient of 76 MB, few rows a group
                                       ([9000], 64, 4104)])                 # y of 74 MB, one group
def test_grouped_mm_results_past_the_caches(dtype, sizes, K, N):
    check_grouped(randn((sum(sizes), K), dtype, 1), randn((len(sizes), K, N), dtype, 2), offsets_of(sizes))


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_mm_rows_of_no_group(dtype):
    """Rows before the first and behind the last group hold infinities and NaN: they reach nothing, and come out zero."""
    x = randn((300, 64), dtype, 3)
    x[:7], x[290:] = math.inf, math.nan
    y, dx, dw = check_grouped(x, randn((3, 64, 72), dtype, 4), offsets_of([100, 0, 183], first=7))
    for t in (y, dx):
        assert float(t[:7].abs().sum()) == 0.0 and float(t[290:].abs().sum()) == 0.0
    assert bool(torch.isfinite(dw).all())
    check_grouped(randn((50, 64), dtype, 3), randn((2, 64, 8), dtype, 4), offsets_of([0, 0], first=20))   # nobody at all


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_mm_infinities_stay_in_their_group(dtype):
    x = randn((200, 128), dtype, 5)
    x[100:] = math.nan      # the second group's rows: in tiles and contractions next to the first group's
    w = randn((2, 128, 64), dtype, 6).requires_grad_(True)
    o = offsets_of([100, 100])
    y = F.grouped_mm(x, w, o)
    assert bool(torch.isfinite(y[:100]).all()) and bool(y[100:].isnan().all())
    dw, = torch.autograd.grad(y, (w,), torch.ones_like(y))
    assert bool(torch.isfinite(dw[0]).all()) and bool(dw[1].isnan().all())


def test_grouped_mm_fp32_is_the_cmodel_chain():
    """fp32 products are the c-model's, bit for bit, forward and backward."""
    sizes, K, N = [70, 0, 129, 31], 100, 90
    x, w, o = randn((230, K), torch.float32, 7).requires_grad_(True), randn((4, K, N), torch.float32, 8).requires_grad_(True), offsets_of(sizes)
    y = F.grouped_mm(x, w, o)
    dy = randn(y.shape, y.dtype, 9)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    at = 0
    for g, n in enumerate(sizes):
        xs, ws, ds = x.detach()[at:at + n].clone(), w.detach()[g].clone(), dy[at:at + n].clone()
        if n:
            assert torch.equal(y.detach()[at:at + n], simple.mm(xs, ws))
            assert torch.equal(dx[at:at + n], simple.mm(ds, ws.t()))
            assert torch.equal(dw[g], simple.mm(xs.t(), ds))
        else:
            assert float(dw[g].abs().sum()) == 0.0
        at += n


def test_grouped_mm_strides_types_and_needs(front):
    o = offsets_of([10, 20, 3], dtype=torch.int64)
    wide = randn((33, 128), torch.bfloat16, 1)
    check_grouped(wide[:, ::2], randn((3, 64, 40), torch.bfloat16, 2), o)                              # x not contiguous
    check_grouped(wide[:, :64], randn((3, 40, 128), torch.bfloat16, 2)[:, :, ::2].transpose(1, 2), o)   # nor weight
    flat = randn((1 + 33 * 64,), torch.float16, 3)
    check_grouped(flat[1:].view(33, 64), randn((1 + 3 * 64 * 40,), torch.float16, 4)[1:].view(3, 64, 40), o)   # odd addresses
    x, w = randn((33, 64), torch.float32, 5), randn((3, 64, 40), torch.float32, 6)
    full = check_grouped(x, w, o)
    y = F.grouped_mm(x.requires_grad_(True), w, o)                                                      # only x, only weight
    assert torch.equal(torch.autograd.grad(y, (x,), randn(y.shape, y.dtype, 11))[0], full[1])
    y = F.grouped_mm(x.detach(), w.requires_grad_(True), o)
    assert torch.equal(torch.autograd.grad(y, (w,), randn(y.shape, y.dtype, 11))[0], full[2])
    y = F.grouped_mm(x, w, o)
    y.sum().backward()                                                                                  # a broadcast gradient
    close(x.grad[:10], (w.detach()[0].double().sum(1))[None].expand(10, 64).clone(), 64 * 64 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("given", TYPES)
def test_grouped_linear_under_autocast(dtype, given, front):
    """fp32 master weights, activations of any type: cast to autocast's type, as torch.nn.Linear does beside it."""
    from mpemu.module_wrappers import GroupedLinear, GroupedMatmul
    layer, lin, o = GroupedLinear(3, 40, 24, device=DEV), torch.nn.Linear(40, 24, device=DEV), offsets_of([10, 0, 21])
    x = randn((31, 40), given, 1).requires_grad_(True)
    dy = randn((31, 24), dtype, 2)
    with torch.autocast("cuda", dtype=dtype):
        y = layer(x, o)
        assert y.dtype == lin(x).dtype == dtype
        got = torch.autograd.grad(y, (x, layer.weight), dy)
        assert torch.equal(GroupedMatmul()(x, layer.weight.transpose(1, 2), o), y)
        with torch.no_grad():
            assert torch.equal(layer(x, o), y)
        with torch.autocast("cuda", enabled=False):
            assert F.grouped_mm(x.float(), layer.weight.transpose(1, 2), o).dtype == torch.float32
    a, w = x.detach().to(dtype).requires_grad_(True), layer.weight.detach().to(dtype).requires_grad_(True)
    want = F.grouped_mm(a, w.transpose(1, 2), o)
    assert torch.equal(y, want)
    for g, t, d in zip(got, (x, layer.weight), torch.autograd.grad(want, (a, w), dy)):
        assert g.dtype == t.dtype and torch.equal(g, d.to(t.dtype))


def test_grouped_mm_gradient_against_differences():
    x, w, o = randn((5, 3), torch.float32, 1).requires_grad_(True), randn((2, 3, 4), torch.float32, 2).requires_grad_(True), offsets_of([2, 3])
    v = randn((5, 4), torch.float32, 3)
    dx, dw = torch.autograd.grad((F.grouped_mm(x, w, o) * v).sum(), (x, w))

    def f(a, b):
        return float((F.grouped_mm(a, b, o).double() * v.double()).sum())

    with torch.no_grad():
        for t, d, at in ((x, dx, (1, 2)), (x, dx, (4, 0)), (w, dw, (0, 1, 3)), (w, dw, (1, 2, 0))):
            e = torch.zeros_like(t)
            e[at] = 0.5
            up, down = (f(x + e, w), f(x - e, w)) if t is x else (f(x, w + e), f(x, w - e))
            assert abs((up - down) - float(d[at])) < 64 * 2.0 ** -22


def test_grouped_mm_refusals(front):
    x, w, o = randn((6, 8), torch.float32, 1), randn((2, 8, 4), torch.float32, 2), offsets_of([2, 4])
    for bad in (lambda: F.grouped_mm(x[0], w, o), lambda: F.grouped_mm(x, w[0], o), lambda: F.grouped_mm(x[:, :7], w, o),
                lambda: F.grouped_mm(x, w, o[:2]), lambda: F.grouped_mm(x, w[:0], o[:1]), lambda: F.grouped_mm(x, w, o[None])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        F.grouped_mm(x.half(), w, o)
    with pytest.raises(RuntimeError):
        y = F.grouped_mm(x.requires_grad_(True), w.requires_grad_(True), o)
        g, = torch.autograd.grad(y.sum(), (x,), create_graph=True)
        torch.autograd.grad(g.sum(), (w,))


# ---- norm and clipping --------------------------------------------------------------------------------------------------------
def norm_reference(grads, p):
    flat = torch.cat([g.detach().double().reshape(-1) for g in grads] + [torch.zeros(1, dtype=torch.float64, device=DEV)])
    return float(flat.abs().max()) if p == math.inf else float(flat.abs().sum()) if p == 1.0 else float(flat.square().sum().sqrt())


def check_clip(grads, max_norm, p, out=None):
    want = norm_reference(grads, p)
    coef = min(1.0, max_norm / (want + 1e-6))
    values = [g.detach().double() * coef for g in grads]
    assert abs(float(F.grad_norm(grads, p)) - want) <= want * 2.0 ** -23 + 2.0 ** -149
    norm = F.clip_grads_(grads, max_norm, norm_type=p, out=out)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= want * 2.0 ** -23 + 2.0 ** -149
    for got, v in zip(grads if out is None else out, values):
        close(got, v, v.abs() * 2.0 ** -21)    # norm, its sum with 1e-6, the quotient and the product: a rounding each
    return norm


SHAPES = [(1000, 77), (1,), (16384,), (16385,), (3, 5, 7), (0,), (40000,), (129,)]


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("share", [0.3, 2.0])
def test_clip_in_place(p, dtype, share, front):
    grads = [randn(s, dtype, i, 0.01) for i, s in enumerate(SHAPES)]
    before = [g.clone() for g in grads]
    check_clip(grads, norm_reference(grads, p) * share, p)
    if share > 1.0:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("share", [0.3, 2.0])
def test_clip_into_master_gradients(dtype, share, front):
    """16-bit gradients into fp32 ones, both views of flat buffers at odd addresses, types mixed within the list."""
    n = sum(math.prod(s) for s in SHAPES)
    sizes = [math.prod(s) for s in SHAPES]
    flat, master = randn((n + 1,), dtype, 1, 0.01)[1:], torch.full((n + 1,), 7.0, device=DEV)[1:]
    grads = [t.view(s) for t, s in zip(flat.split(sizes), SHAPES)] + [randn((500,), torch.float32, 2, 0.01)]
    outs = [t.view(s) for t, s in zip(master.split(sizes), SHAPES)] + [torch.empty(500, device=DEV)]
    before = flat.clone()
    check_clip(grads, norm_reference(grads, 2.0) * share, 2.0, out=outs)
    assert torch.equal(flat, before)


def test_clip_many_tensors(front):
    """More tensors than one launch's table holds, and a list of nothing but empty ones."""
    grads = [randn((1 + 37 * i % 301,), (torch.float32, torch.bfloat16, torch.float16)[i % 3], i, 0.1) for i in range(400)]
    check_clip(grads, 1.0, 2.0)
    assert float(F.clip_grads_([torch.zeros(0, device=DEV)] * 3, 1.0)) == 0.0


def test_clip_large_and_small_values():
    big = [torch.full((1000,), 3.0e38, device=DEV), torch.full((70,), -3.0e38, device=DEV)]
    check_clip(big, 1.0e38, math.inf)
    small = [torch.full((100000,), 1.0e-30, device=DEV)]     # squares below fp32's range
    check_clip(small, 1.0, 2.0)
    many = [torch.full((1 << 24,), 1.0, device=DEV), torch.full((1 << 20,), 1.0e-4, device=DEV)]
    check_clip(many, 3.0, 1.0)
    check_clip([torch.zeros(50, device=DEV)], 1.0, 2.0)
    check_clip([torch.ones(50, device=DEV)], 0.0, 2.0)


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_clip_not_finite(p, front):
    g = [torch.ones(100, device=DEV), torch.ones(70000, device=DEV)]
    g[1][69999] = math.nan
    kept = [t.clone() for t in g]
    with pytest.raises(RuntimeError):
        F.clip_grads_(g, 1.0, p, error_if_nonfinite=True)
    assert all(torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) for a, b in zip(g, kept))   # as they were
    assert math.isnan(float(F.clip_grads_(g, 1.0, p))) and bool(g[0].isnan().all())
    g = [torch.ones(100, device=DEV), torch.full((3,), -math.inf, device=DEV)]
    assert float(F.clip_grads_(g, 1.0, p)) == math.inf
    assert float(g[0].abs().sum()) == 0.0 and bool(g[1].isnan().all())                       # inf * 0, as torch


FOURS = {   # eight neighbours: two fours whose squares are added in fp32 where its range holds them, in 64 bits where not
    torch.bfloat16: [[1e30] * 8, [1e-30] * 8, [1e30] * 4 + [0.0] * 4, [0.0] * 4 + [1e-30] * 4, [1e-30] * 4 + [1.0] * 4,
                     [1.0] * 4 + [1e-38] * 4, [1e-39, 0, 0, 0, 0, 0, 1e-39, 0], [3e38, 0, 0, 0, 0, 0, 0, 0], [1e-20, 1e10, 3.0, 0, 0, 0, -7.0, 0],
                     [2.0 ** -45] * 8, [2.0 ** -46] * 8, [0.75 * 2.0 ** -44, 0, 0, 0] * 2, [2.0 ** 61] * 8, [2.0 ** 61.5] * 8,
                     [2.0 ** 63, 0, 0, 0, 1.0, 0, 0, 0], [1.9 * 2.0 ** 63, 0, 0, 0, 0, 0, 0, 2.0 ** -60]],
    torch.float16: [[65504.0] * 8, [2.0 ** -24] * 8, [65504.0] * 4 + [0.0] * 4, [0.0] * 4 + [2.0 ** -24] * 4,
                    [2.0 ** -24] * 4 + [65504.0] * 4, [2.0 ** -24, 0, 0, 0, 0, 0, 0, 0], [0.0] * 7 + [-60000.0], [2.0 ** -14, 6e-8, 1.0, -3e4] * 2]}


@pytest.mark.parametrize("dtype,eight", [(t, e) for t in SIXTEEN for e in FOURS[t]])
@pytest.mark.parametrize("repeat,tail", [(1, 0), (1, 5), (130, 3), (3000, 7)])
def test_norm_of_16_bit_values_over_their_range(dtype, eight, repeat, tail):
    """Squares beyond fp32's range, below it, and beside zeros.  A four's sum is off by two roundings, 2^-23 at most, its root
    by half of that; the norm is rounded once more, 2^-24."""
    values = (eight * (repeat + 1))[:8 * repeat + tail]
    g = torch.tensor(values, dtype=torch.float64, device=DEV).to(dtype)
    for p in (1.0, 2.0, math.inf):
        want = norm_reference([g], p)
        got = float(F.grad_norm([g], p))
        if want >= 2.0 ** 128 * (1 - 2.0 ** -25):   # rounds to infinity
            assert got == math.inf
        else:
            assert abs(got - want) <= want * (2.0 ** -23 + 2.0 ** -40) + 2.0 ** -150, (p, got, want)
    want = norm_reference([g], 2.0)
    if want < 2.0 ** 127:
        limit = torch.tensor(0.3 * want).item()
        coef = min(1.0, limit / (want + 1e-6))
        v = g.double() * coef
        F.clip_grads_([g], limit)
        close(g, v, v.abs() * 2.0 ** -21)


@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("at", [0, 5, 4001, 9999])
def test_clip_of_16_bit_values_not_finite(p, dtype, at, front):
    g = torch.ones(10001, device=DEV, dtype=dtype)
    g[at] = math.nan
    kept = g.clone()
    with pytest.raises(RuntimeError, match="norm of the gradients"):
        F.clip_grads_([g], 1.0, p, error_if_nonfinite=True)
    assert torch.equal(g.nan_to_num(5.0), kept.nan_to_num(5.0))
    assert math.isnan(float(F.grad_norm([g], p)))
    g[at] = -math.inf
    assert float(F.clip_grads_([g], 1.0, p)) == math.inf
    assert bool(g[at].isnan()) and float(g.nan_to_num(0.0).abs().sum()) == 0.0    # inf * 0, as torch
    g = torch.ones(10001, device=DEV, dtype=dtype)
    g[at], g[(at + 1) % 10001] = math.inf, math.nan
    assert math.isnan(float(F.clip_grads_([g], 1.0, p))) and bool(g.isnan().all())


def test_clip_layouts_and_overlap(front):
    conv = randn((8, 6, 3, 3), torch.float32, 1).contiguous(memory_format=torch.channels_last)
    strided = randn((40, 30), torch.float32, 2)
    rest = strided.clone()
    check_clip([conv, strided[:, ::2]], 0.5, 2.0)
    assert torch.equal(strided[:, 1::2], rest[:, 1::2])
    t = randn((100,), torch.float32, 3)
    for grads, out in (([t, t], None), ([t[:60], t[50:]], None), ([t[:1].expand(9)], None), ([t[:50], t[50:]], [t[50:], torch.empty(50, device=DEV)])):
        keep = t.clone()
        with pytest.raises(ValueError):
            F.clip_grads_(grads, 1.0, out=out)
        assert torch.equal(t, keep)
    for grads, out in (([t], [t, t]), ([t], [t[:50]]), ([t], [t.half()])):
        with pytest.raises(ValueError):
            F.clip_grads_(grads, 1.0, out=out)


def test_clip_refuses_shared_memory_in_gradients_with_gaps(front):
    """Gradients that do not fill their memory are copied on their way: their own addresses count all the same."""
    s, line = randn((40, 30), torch.float32, 2), randn((64,), torch.float32, 3)
    kept = s.clone(), line.clone()
    for grads in ([s[:, ::2], s], [s[:, ::2], s[:, ::2]], [line.as_strided((4, 4), (2, 1))], [s[:, :11], s[:, 10:]]):
        with pytest.raises(ValueError, match="shares memory"):
            F.clip_grads_(grads, 0.5)
        assert torch.equal(s, kept[0]) and torch.equal(line, kept[1])
    check_clip([s[:, 1::2], s[:, ::2]], 0.5, 2.0)     # side by side
    check_clip([s[:, :10], s[:, 10:]], 0.1, 2.0)


def test_clip_moves_the_version(front):
    """A gradient that autograd still needs must not change unseen."""
    a = randn((10,), torch.float32, 1).requires_grad_(True)
    g = randn((10,), torch.float32, 2)
    kept, out = (a * g).sum(), torch.empty(10, device=DEV)
    F.clip_grads_([g], 0.1, out=[out])
    before = out._version
    F.clip_grads_([randn((10,), torch.float32, 2)], 0.1, out=[out])
    assert out._version > before
    F.clip_grads_([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        kept.backward()


def test_clip_over_a_group_of_one(front, tmp_path):
    """The sharded form through a process group: gloo stages the one word through the host."""
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method="file://" + str(tmp_path / "store"), rank=0, world_size=1)
    try:
        for p in (1.0, 2.0, math.inf):
            g = [randn((1000,), torch.bfloat16, 1), randn((77,), torch.float32, 2)]
            twin = [t.clone() for t in g]
            a, b = F.clip_grads_(g, 0.5, p, group=dist.group.WORLD), F.clip_grads_(twin, 0.5, p)
            assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(g, twin))
        assert float(F.clip_grads_([], 1.0, group=dist.group.WORLD)) == 0.0
    finally:
        dist.destroy_process_group()


def _one_rank_rccl(rank, store, out):
    import os
    import sys
    import torch.distributed as dist
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp8-emulation-toolkit_amd"))
    from mpemu import functional
    from mpemu.sharded import group_backend
    dev = torch.device("cuda", 0)
    torch.cuda.set_device(dev)
    dist.init_process_group("nccl", init_method="file://" + store, rank=0, world_size=1, device_id=dev)
    assert group_backend() == "nccl"
    same = []
    for p in (1.0, 2.0, math.inf):
        for odd in (1.0, math.inf, math.nan):
            g = [torch.linspace(-3, 2, 1000, device=dev).bfloat16(), torch.full((77,), 0.5, device=dev)]
            g[1][5] = odd
            twin = [t.clone() for t in g]
            a, b = functional.clip_grads_(g, 0.5, p, group=dist.group.WORLD), functional.clip_grads_(twin, 0.5, p)
            same += [torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0)) and torch.equal(x.isnan(), y.isnan())
                     for x, y in zip([a] + g, [b] + twin)]
    same.append(float(functional.clip_grads_([], 1.0, group=dist.group.WORLD)) == 0.0)
    torch.save(same, out)
    dist.destroy_process_group()


def test_clip_over_an_rccl_group_of_one(tmp_path):
    """The branch that reduces the word on the device, through a communicator of one rank."""
    store, out = str(tmp_path / "store"), str(tmp_path / "out")
    torch.multiprocessing.spawn(_one_rank_rccl, args=(store, out), nprocs=1)
    same = torch.load(out, weights_only=True)
    assert len(same) == 28 and all(same), same


@pytest.mark.parametrize("sharded", [False, True])
def test_clip_refuses_a_norm_beyond_float32(front, sharded, tmp_path):
    """Four times 3e38: the 64-bit sum is finite, the norm (6e38) is not a float32; 4e19: the sum of squares is not one, the norm is."""
    import torch.distributed as dist
    group = None
    if sharded:
        dist.init_process_group("gloo", init_method="file://" + str(tmp_path / "store"), rank=0, world_size=1)
        group = dist.group.WORLD
    try:
        g = torch.full((4,), 3e38, device=DEV)
        with pytest.raises(RuntimeError, match="norm of the gradients is inf"):
            F.clip_grads_([g], 1.0, error_if_nonfinite=True, group=group)
        assert torch.equal(g, torch.full((4,), 3e38, device=DEV))
        g = torch.full((4,), 4e19, device=DEV)
        norm = F.clip_grads_([g], 1.0, error_if_nonfinite=True, group=group)
        assert abs(float(norm) - 8e19) <= 8e19 * 2.0 ** -22
        close(g, torch.full((4,), 0.5, dtype=torch.float64, device=DEV), 0.5 * 2.0 ** -21)
    finally:
        if sharded:
            dist.destroy_process_group()


def test_clip_grad_norm_of_parameters(front):
    ps = [torch.nn.Parameter(randn((50, 20), torch.float32, i)) for i in range(4)]
    for p in ps[:3]:
        p.grad = randn(p.shape, p.dtype, 9)
    twin = [p.grad.clone() for p in ps[:3]]
    norm = F.clip_grad_norm_(iter(ps), 1.5)
    want = norm_reference(twin, 2.0)
    assert abs(float(norm) - want) <= want * 2.0 ** -23 and ps[3].grad is None
    for p, t in zip(ps, twin):
        v = t.double() * (1.5 / (want + 1e-6))
        close(p.grad, v, v.abs() * 2.0 ** -21)


# ---- beyond 32 bits, and nothing at all --------------------------------------------------------------------------------------------
def test_addresses_beyond_32_bits():
    """Tables, rows and gradients of more than 2^31 elements (over 4 GB): the last ones are read and written where they are."""
    vocab, width = (1 << 20) + 7, 2056
    table = torch.zeros((vocab, width), dtype=torch.bfloat16, device=DEV)
    ids = torch.tensor([vocab - 1, 0, vocab - 1, 1 << 20, vocab, 5], device=DEV)
    table[ids[ids < vocab]] = randn((5, width), torch.bfloat16, 1)
    table.requires_grad_(True)
    out = F.embedding(ids, table, scale=2.0)
    assert torch.equal(out[[0, 1, 2, 3, 5]], table.detach()[ids[[0, 1, 2, 3, 5]]] * 2.0) and bool(out[4].isnan().all())
    dout = randn(out.shape, out.dtype, 2)
    dt, = torch.autograd.grad(out, (table,), dout)
    for v in (0, 5, 1 << 20, vocab - 1):
        want = dout[ids == v].double().sum(0) * 2.0
        close(dt[v], want, dout[ids == v].double().abs().sum(0) * 2.0 * 4 * 2.0 ** -24)
    assert int(dt.count_nonzero()) == int(dt[[0, 5, 1 << 20, vocab - 1]].count_nonzero())
    del out
    norm = F.clip_grads_([dt], 0.5)
    want = norm_reference([dt[[0, 5, 1 << 20, vocab - 1]]], 2.0)     # now clipped to 0.5; each element rounded to bf16, a few times fp32
    assert abs(want - 0.5) <= 0.5 * (2.0 ** -8 + 2.0 ** -20) and float(norm) > 0.5
    # the same memory as rows of a product: the last group lies behind 4 GB
    x, w = table.detach(), randn((3, width, 40), torch.bfloat16, 3).requires_grad_(True)
    first = vocab - 300
    o = torch.tensor([7, first - 1000, first, vocab - 1], dtype=torch.int32, device=DEV)
    y = F.grouped_mm(x.requires_grad_(True), w, o)
    dy = randn(y.shape, y.dtype, 4)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    X, W, DY = x.detach()[first:vocab - 1].double(), w.detach()[2].double(), dy[first:vocab - 1].double()
    close(y.detach()[first:vocab - 1], X @ W, (X.abs() @ W.abs()) * ((width + 1) * 2.0 ** -23))
    close(dx[first:vocab - 1], DY @ W.t(), (DY.abs() @ W.t().abs()) * (41 * 2.0 ** -23))
    close(dw[2], X.t() @ DY, (X.t().abs() @ DY.abs()) * (300 * 2.0 ** -23))
    assert float(y.detach()[vocab - 1].abs().sum()) == 0.0 and float(dx[vocab - 1].abs().sum()) == 0.0 and float(dx[:7].abs().sum()) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
def test_no_columns_at_all(dtype, front):
    """An empty contraction is zero; no columns are no results."""
    o = offsets_of([2, 3])
    for k, n in ((0, 8), (0, 5), (8, 0), (0, 0)):
        x, w = torch.ones(6, k, dtype=dtype, device=DEV, requires_grad=True), torch.ones(2, k, n, dtype=dtype, device=DEV, requires_grad=True)
        y = F.grouped_mm(x, w, o)
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert y.shape == (6, n) and float(y.detach().abs().sum()) == float(dx.abs().sum()) == float(dw.abs().sum()) == 0.0
        assert dx.shape == x.shape and dw.shape == w.shape
    table = torch.ones(4, 0, dtype=dtype, device=DEV, requires_grad=True)
    out = F.embedding(torch.tensor([1, 9], device=DEV), table)
    assert out.shape == (2, 0) and torch.autograd.grad(out, (table,), torch.ones_like(out))[0].shape == (4, 0)


# ---- streams, capture, repetition -------------------------------------------------------------------------------------------------
def _step(ids, experts, table, w, o_rows):
    order, offsets = F.group_rows(experts, w.shape[0])
    h = F.embedding(ids, table, scale=2.0)
    y = F.grouped_mm(h.index_select(0, order), w, offsets)
    dt, dw = torch.autograd.grad(y, (table, w), torch.ones_like(y))
    norm = F.clip_grads_([dt, dw], 0.5)
    return [y.detach(), dt, dw, norm, order, offsets]


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_and_on_other_streams(dtype):
    """A whole step in a HIP graph, replayed on new inputs with eager work between the replays, and on a side stream: the
    eager results, bit for bit (every sum has one order)."""
    def inputs(seed):
        return (torch.randint(0, 500, (6000,), generator=gen(seed), device=DEV), torch.randint(0, 9, (6000,), generator=gen(seed + 1), device=DEV))

    table, w = randn((500, 64), dtype, 1).requires_grad_(True), randn((9, 64, 96), dtype, 2, 0.1).requires_grad_(True)
    ids, experts = inputs(1)
    eager = [t.clone() for t in _step(ids, experts, table, w, None)]
    again = _step(ids, experts, table, w, None)
    assert all(torch.equal(a, b) for a, b in zip(eager, again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _step(ids, experts, table, w, None)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graphs = []
    for _ in range(2):      # two graphs alive at once share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(ids, experts, table, w, None)
        graphs.append((g, out))
    for seed in (1, 5, 9, 1):
        a, b = inputs(seed)
        ids.copy_(a), experts.copy_(b)
        want = [t.clone() for t in _step(ids, experts, table, w, None)]
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, want)), seed


@pytest.mark.parametrize("held", ["table", "weight", "view"])
def test_captured_backward_beside_a_live_eager_graph(held, front):
    """A capture whose leaves an eager graph still holds would end the process at its backward pass: refused at the forward
    call, and fine once the eager graph is gone."""
    table = randn((50, 16), torch.float32, 1).requires_grad_(True)
    w, o = randn((2, 8, 16), torch.float32, 2).requires_grad_(True), offsets_of([10, 20])
    ids = torch.randint(0, 50, (30,), generator=gen(3), device=DEV)

    def step():
        if held == "table":
            return F.embedding(ids, table)
        x = F.embedding(ids, table.detach())
        return F.grouped_mm(x, w.transpose(1, 2) if held == "view" else w.view(2, 16, 8), o)

    alive = step()
    want = torch.autograd.grad(alive, (table if held == "table" else w,), torch.ones_like(alive), retain_graph=True)[0]
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    torch.cuda.synchronize()
    if front == "ctypes":
        return
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
        got, = torch.autograd.grad(y, (table if held == "table" else w,), torch.ones_like(y))
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


# ---- together, as a model uses them -------------------------------------------------------------------------------------------------
class Experts(torch.nn.Module):
    """A small language model with experts: scaled embedding, a router, grouped products, a head."""

    def __init__(self, vocab=97, d=64, ff=96, groups=5, top=2):
        super().__init__()
        from mpemu.module_wrappers import GroupedLinear, ScaledEmbedding
        self.groups, self.top = groups, top
        self.embeddings = ScaledEmbedding(vocab, d, padding_idx=0, scale=8.0)
        self.router = torch.nn.Linear(d, groups)
        self.up, self.down = GroupedLinear(groups, d, ff), GroupedLinear(groups, ff, d)
        self.head = torch.nn.Linear(d, vocab)

    def forward(self, ids):
        h = self.embeddings(ids).reshape(-1, self.embeddings.embedding_dim)
        gate, choice = self.router(h).softmax(-1).topk(self.top, -1)
        order, offsets = F.group_rows(choice, self.groups)
        token = order.long() // self.top
        e = self.down(torch.relu(self.up(h[token], offsets)), offsets) * gate.reshape(-1)[order.long()].unsqueeze(1)
        return self.head(h + torch.zeros_like(h).index_add(0, token, e))

    def plain(self, ids, dtype=torch.float64):
        p = {k: v.detach().to(dtype).requires_grad_(True) for k, v in self.named_parameters()}
        h = p["embeddings.weight"][ids.reshape(-1)] * 8.0
        gate, choice = (h @ p["router.weight"].t() + p["router.bias"]).softmax(-1).topk(self.top, -1)
        out = h
        for k in range(self.top):
            a = torch.relu((p["up.weight"][choice[:, k]] @ h.unsqueeze(2)).squeeze(2))
            out = out + (p["down.weight"][choice[:, k]] @ a.unsqueeze(2)).squeeze(2) * gate[:, k:k + 1]
        return out @ p["head.weight"].t() + p["head.bias"], p


def test_model_with_experts_trains():
    torch.manual_seed(3)
    model = Experts().to(DEV)
    ids = torch.randint(1, 97, (4, 50), generator=gen(1), device=DEV)
    ids[:, 45:] = 0
    target = torch.randint(0, 97, (200,), generator=gen(2), device=DEV)
    torch.nn.functional.cross_entropy(model(ids), target).backward()
    logits, p = model.plain(ids)
    torch.nn.functional.cross_entropy(logits, target).backward()
    for name, q in model.named_parameters():
        want = p[name].grad
        if name == "embeddings.weight":
            want[0] = 0.0
        assert float((q.grad.double() - want).norm()) <= 1e-5 * float(want.norm()), name   # fp32, a dozen layers of sums of < 200 terms
    norm = F.clip_grad_norm_(model.parameters(), 0.1)
    total = math.sqrt(sum(float(q.grad.double().square().sum()) for q in model.parameters()))
    assert float(norm) > 0.1 and abs(total - 0.1) < 1e-5


@pytest.mark.parametrize("algo", ["hybrid", "direct"])
def test_model_with_experts_trains_emulated(algo):
    """The same under the emulators: hooks on the new modules, gradients clipped in optimizer_step, master weights on the
    FP16 grid, and what the experts receive on the FP8 grid."""
    from mpemu import mpt_emu
    torch.manual_seed(4)
    model = Experts().to(DEV).train()
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    model, emu = mpt_emu.initialize(model, opt, training_algo=algo, device=DEV, list_exempt_layers=["head", "router"])
    seen = []
    model.up.register_forward_pre_hook(lambda m, a: seen.append((a[0].detach().clone(), a[1].clone())))
    ids = torch.randint(1, 97, (4, 50), generator=gen(1), device=DEV)
    target = torch.randint(0, 97, (200,), generator=gen(2), device=DEV)
    for _ in range(2):
        opt.zero_grad()
        torch.nn.functional.cross_entropy(model(ids), target).backward()
        raw = norm_reference([q.grad for q in model.parameters()], 2.0)
        norm = emu.optimizer_step(opt, max_grad_norm=0.05)
        assert abs(float(norm) - raw) <= raw * 2.0 ** -23
        now = norm_reference([q.grad for q in model.parameters()], 2.0)
        assert now <= max(raw, 0.05) and abs(now - min(raw, 0.05)) < 1e-5
        for q in model.parameters():
            assert bool(torch.isfinite(q).all()) and torch.equal(q.detach(), q.detach().half().float())
    x, offsets = seen[0]
    assert offsets.dtype == torch.int32 and int(offsets[-1]) == 400
    assert len(x.unique()) < 600                        # 8-bit values
    assert emu.optimizer_step(opt) is None


def test_model_with_experts_quantised_for_inference():
    """Post-training quantisation: one scale per expert under per-channel scaling, the table's rows likewise."""
    from mpemu import mpt_emu, qutils
    torch.manual_seed(5)
    model = Experts().to(DEV).eval()
    up, table = model.up.weight.detach().clone(), model.embeddings.weight.detach().clone()
    model, _ = mpt_emu.quantize_model(model, dtype="e4m3", device=DEV)
    cfg = qutils.TensorQuantConfig("e4m3", "rne", "per-channel")
    for g in range(5):
        one = qutils.quantize_tensor(up[g:g + 1].contiguous(), cfg, None)
        assert torch.equal(model.up.weight[g:g + 1].detach(), one)
    assert torch.equal(model.embeddings.weight.detach(), qutils.quantize_tensor(table, cfg, None))
    with torch.no_grad():
        assert bool(torch.isfinite(model(torch.randint(0, 97, (2, 3), device=DEV))).all())


def test_abi_of_the_front():
    assert hip.ext() is not None and hip.ext().abi_version() == hip.lib().fpemu_abi_version() == 11
