"""Tokens sorted by expert and back, and the gradients, against the definitions.

Bounds.  Rows and orders are equal exactly.  A sum of n fp32 products has an error of at most
(n + 1) * 2^-24 of the sum of their magnitudes, and its rounding to type t eps(t) / 2 of the value.
A weight's gradient is a dot product over H, 256 threads' partial sums of at most H / 256 + 8
terms and a tree of 5 + 8 more.
"""
import math

import pytest
import torch

gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def plain_order(idx, E, first=0):
    T, K = idx.shape
    flat = idx.reshape(-1).tolist()
    of = [[] for _ in range(E)]
    for i, e in enumerate(flat):
        if e >= 0 and 0 <= e - first < E:
            of[e - first].append(i)
    route = [i for e in of for i in e]
    offsets = [0]
    for e in of:
        offsets.append(offsets[-1] + len(e))
    row_of = [-1] * (T * K)
    for r, i in enumerate(route):
        row_of[i] = r
    return (torch.tensor(row_of, dtype=torch.int32).view(T, K),
            torch.tensor(route + [-1] * (T * K - len(route)), dtype=torch.int32),
            torch.tensor(offsets, dtype=torch.int32))


def make_idx(T, K, E, absent=0.2, seed=0, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, max(E, 1), (T, K), generator=g)
    idx = torch.where(torch.rand(T, K, generator=g) < absent, torch.full_like(idx, -1), idx)
    return idx.to(dtype)


def order_of(idx, E, **kw):
    from constellation_b200.token_sort import sort_routes

    return sort_routes(idx.cuda(), E, **kw)


def same_order(o, idx, E, first=0):
    for got, want in zip((o.row_of, o.route_of, o.offsets), plain_order(idx, E, first)):
        assert torch.equal(got.cpu(), want)


@gpu
@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (1, 8, 256), (3, 2, 5), (64, 8, 256), (500, 8, 1024), (511, 8, 7),
                                   (513, 8, 64), (1000, 3, 33), (4096, 8, 256), (20000, 1, 2), (5, 1024, 1024)])
def test_orders(T, K, E):
    idx = make_idx(T, K, E, seed=T)
    same_order(order_of(idx, E), idx, E)


@gpu
@pytest.mark.parametrize("T", [1, 40, 3000])
def test_orders_at_the_edges(T):
    E = 16
    for idx in (torch.full((T, 4), -1, dtype=torch.int32), torch.full((T, 4), E, dtype=torch.int32),
                torch.full((T, 4), 3, dtype=torch.int32), torch.full((T, 4), -2 ** 31, dtype=torch.int32),
                torch.full((T, 4), 2 ** 31 - 1, dtype=torch.int32)):
        same_order(order_of(idx, E), idx, E)
    wide = make_idx(T, 4, 100, seed=1, dtype=torch.int64)
    same_order(order_of(wide, E), wide, E)
    same_order(order_of(wide, E, first_expert=32), wide, E, 32)
    far = torch.tensor([[2 ** 40 + 1, -2 ** 40, 1, 2 ** 32 + 2]]).repeat(T, 1)
    same_order(order_of(far, E), far, E)
    same_order(order_of(wide.t().contiguous().t(), E), wide, E)


@gpu
def test_no_tokens():
    from constellation_b200.token_sort import sort_tokens, unsort_tokens

    o = order_of(torch.zeros((0, 8), dtype=torch.int32), 5)
    assert o.offsets.tolist() == [0] * 6 and o.row_of.shape == (0, 8)
    rows = sort_tokens(torch.zeros(0, 64, device="cuda"), o)
    assert rows.shape == (0, 64)
    assert unsort_tokens(rows, o, torch.zeros(0, 8, device="cuda")).shape == (0, 64)


def rand(shape, dt, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to("cuda", dt)


@gpu
@pytest.mark.parametrize("dt", DTYPES + [torch.float8_e4m3fn])
@pytest.mark.parametrize("H", [1, 3, 8, 100, 127, 2048, 5001, 7168])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 8), (70, 6)])
def test_sorted_rows(T, K, H, dt):
    from constellation_b200.token_sort import sort_tokens

    E = 16
    idx = make_idx(T, K, E, seed=H)
    o = order_of(idx, E)
    x = rand((T, H), torch.float32, 1).to(dt)
    used = int(o.offsets[-1])
    route = o.route_of[:used].long()
    bits = torch.uint8 if dt == torch.float8_e4m3fn else dt
    want = torch.zeros(T * K, H, dtype=bits, device="cuda")
    want[:used] = x.view(bits)[route // K]
    assert torch.equal(sort_tokens(x, o).view(bits), want)
    scale = rand((T, (H + 127) // 128), torch.float32, 2)
    rows, s = sort_tokens(x, o, scale=scale)
    assert torch.equal(rows.view(bits), want) and rows.dtype == dt
    assert torch.equal(s[:used], scale[route // K]) and (s[used:] == 0).all()


@gpu
@pytest.mark.parametrize("offset,H,width", [(0, 256, 264), (5, 250, 301), (8, 128, 512)])
def test_strided_tokens(offset, H, width):
    from constellation_b200.token_sort import sort_tokens, unsort_tokens

    T, K, E = 33, 4, 8
    o = order_of(make_idx(T, K, E), E)
    x = rand((T, width), torch.bfloat16, 1)[:, offset:offset + H]
    assert torch.equal(sort_tokens(x, o), sort_tokens(x.contiguous(), o))
    assert torch.equal(sort_tokens(x[:1].expand(T, H), o), sort_tokens(x[:1].repeat(T, 1), o))
    y = rand((T * K, width), torch.bfloat16, 2)[:, offset:offset + H]
    res = rand((T, width), torch.float32, 3)[:, offset:offset + H]
    w = rand((K, T), torch.float32, 4).t()
    assert torch.equal(unsort_tokens(y, o, w, residual=res),
                       unsort_tokens(y.contiguous(), o, w.contiguous(), residual=res.contiguous()))


def plain_unsort(rows, o, w, res):
    T, K = o.row_of.shape
    out = torch.zeros(T, rows.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    for k in range(K):
        t = (o.row_of[:, k] >= 0).nonzero().view(-1)
        r = o.row_of[t, k].long()
        p = rows[r].double() * (1.0 if w is None else w[t, k].double()[:, None])
        out[t] += p
        mag[t] += p.abs()
    if res is not None:
        out += res.double()
        mag += res.double().abs()
    return out, mag


@gpu
@pytest.mark.parametrize("dt,od", [(a, b) for a in DTYPES for b in DTYPES])
@pytest.mark.parametrize("H", [1, 7, 256, 5001, 7168])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 8), (37, 6), (150, 17)])
def test_unsorted_sums(T, K, H, dt, od):
    from constellation_b200.token_sort import unsort_tokens

    E = 16
    o = order_of(make_idx(T, K, E, seed=T + K), E)
    rows, w = rand((T * K, H), dt, 1), rand((T, K), torch.float32, 2)
    rows[int(o.offsets[-1]):] = math.nan  # rows behind the last expert's are not read
    w = torch.where(o.row_of < 0, torch.full_like(w, math.inf), w)  # nor are absent routes' weights
    for weight, res in ((w, None), (None, rand((T, H), dt, 3)), (w, rand((T, H), torch.float32, 4))):
        got = unsort_tokens(rows, o, weight, residual=res, out_dtype=od)
        ref, mag = plain_unsort(rows, o, weight, res)
        bound = (K + 2) * U * mag + ref.abs() * torch.finfo(od).eps / 2 + torch.finfo(od).smallest_normal
        assert got.dtype == od and ((got.double() - ref).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,K,H", [(1, 1, 8), (1, 8, 7168), (37, 6, 255), (300, 8, 1024), (20, 33, 264)])
def test_gradients_follow_the_formulas(T, K, H, dt):
    from constellation_b200.token_sort import (sort_tokens, sort_tokens_backward, unsort_tokens,
                                               unsort_tokens_backward)

    E = 16
    o = order_of(make_idx(T, K, E, seed=T), E)
    used = int(o.offsets[-1])
    half = torch.finfo(dt).eps / 2
    x, g = rand((T, H), dt, 1).requires_grad_(), rand((T * K, H), dt, 2)
    g[used:] = math.nan
    (dx,) = torch.autograd.grad(sort_tokens(x, o), x, g)
    ref, mag = plain_unsort(g, o, None, None)
    assert ((dx.double() - ref).abs() <= (K + 1) * U * mag + half * ref.abs()).all() and dx.dtype == dt
    assert torch.equal(sort_tokens_backward(g, o), dx)

    rows, w = rand((T * K, H), dt, 3).requires_grad_(), rand((T, K), torch.float32, 4).requires_grad_()
    res, go = rand((T, H), torch.float32, 5).requires_grad_(), rand((T, H), dt, 6)
    out = unsort_tokens(rows, o, w, residual=res, out_dtype=dt)
    d_rows, d_w, d_res = torch.autograd.grad(out, (rows, w, res), go)
    assert torch.equal(d_res, go.float())
    route = o.route_of[:used].long()
    want = w.detach().double().view(-1)[route][:, None] * go.double()[route // K]
    assert ((d_rows[:used].double() - want).abs() <= want.abs() * (half + U) + 2.0 ** -25).all()
    assert (d_rows[used:] == 0).all() and d_rows.dtype == dt
    r = o.row_of.clamp(min=0).long()
    prod = rows.detach().double()[r] * go.double()[:, None]
    here = o.row_of >= 0
    bound = (H // 256 + 8 + 14) * U * prod.abs().sum(2)
    assert ((d_w.double() - prod.sum(2)).abs() <= bound)[here].all() and (d_w[~here] == 0).all()
    a, b = unsort_tokens_backward(go, rows, o, w)
    assert torch.equal(a, d_rows) and torch.equal(b, d_w)
    a, b = unsort_tokens_backward(go, rows, o)
    assert b is None and torch.equal(a, sort_tokens(go.to(dt), o))


@gpu
def test_gradients_follow_differences():
    """The map rows, w -> out is linear in each, so a central difference is exact up to rounding."""
    from constellation_b200.token_sort import sort_tokens, unsort_tokens

    T, K, E, H = 9, 3, 4, 40
    o = order_of(make_idx(T, K, E), E)
    x, w = rand((T, H), torch.float32, 1).requires_grad_(), rand((T, K), torch.float32, 2).requires_grad_()
    go = rand((T, H), torch.float32, 3)

    def value(x, w):
        y = sort_tokens(x, o)
        return (unsort_tokens(y, o, w).double() * go.double()).sum()

    dx, dw = torch.autograd.grad(value(x, w), (x, w))
    with torch.no_grad():
        for grad, name in ((dx, "x"), (dw, "w")):
            d = rand(grad.shape, torch.float32, 5)
            a = value(x + d, w) if name == "x" else value(x, w + d)
            b = value(x - d, w) if name == "x" else value(x, w - d)
            want = (grad.double() * d.double()).sum()
            # some thousand rounded terms of magnitude about 1, each off by a few units
            assert abs(float((a - b) / 2 - want)) <= T * H * K * 8 * U * 4


@gpu
def test_partial_gradients_and_unused_inputs():
    from constellation_b200.token_sort import unsort_tokens

    T, K, E, H = 6, 2, 4, 64
    o = order_of(make_idx(T, K, E), E)
    rows, w, go = rand((T * K, H), torch.bfloat16, 1), rand((T, K), torch.float32, 2), rand((T, H), torch.bfloat16, 3)
    both = torch.autograd.grad(unsort_tokens(rows.requires_grad_(), o, w.requires_grad_()), (rows, w), go)
    only = torch.autograd.grad(unsort_tokens(rows, o, w.detach()), rows, go)
    assert torch.equal(only[0], both[0])
    only = torch.autograd.grad(unsort_tokens(rows.detach(), o, w), w, go)
    assert torch.equal(only[0], both[1])
    out = unsort_tokens(rows, o)
    out.sum().backward()  # a gradient with strides of zero
    assert torch.equal(rows.grad[:int(o.offsets[-1])], torch.ones_like(rows[:int(o.offsets[-1])]))


@gpu
def test_repeats_bit_for_bit_and_in_graphs():
    from constellation_b200.token_sort import sort_routes, sort_tokens, sort_tokens_backward, unsort_tokens, \
        unsort_tokens_backward

    T, K, E, H = 700, 8, 64, 1024
    idx, x, w = make_idx(T, K, E).cuda(), rand((T, H), torch.bfloat16, 1), rand((T, K), torch.float32, 2)

    def step(idx, x, w):
        o = sort_routes(idx, E)
        rows = sort_tokens(x, o)
        out = unsort_tokens(rows, o, w)
        return [rows, out, sort_tokens_backward(rows, o), *unsort_tokens_backward(out, rows, o, w)]

    want = step(idx, x, w)
    assert all(torch.equal(a, b) for a, b in zip(step(idx, x, w), want))
    torch.cuda.synchronize()
    other = (idx.flip(0).contiguous(), x.flip(0).contiguous(), w.flip(0).contiguous())
    graphs, held = [], []
    for args in ((idx, x, w), other):  # two graphs alive at once
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(*args))
    want2 = step(*other)
    for g in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held[0], want))
    assert all(torch.equal(a, b) for a, b in zip(held[1], want2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(idx, x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_refusals_of_device_tensors():
    from constellation_b200.token_sort import TokenOrder, sort_routes, sort_tokens, unsort_tokens

    T, K, E, H = 4, 2, 8, 16
    idx = make_idx(T, K, E).cuda()
    o = sort_routes(idx, E)
    x, rows, w = rand((T, H), torch.bfloat16, 1), rand((T * K, H), torch.bfloat16, 2), rand((T, K), torch.float32, 3)
    bad = [lambda: sort_tokens(x[:3], o), lambda: unsort_tokens(rows[:7], o, w), lambda: unsort_tokens(rows, o, w[:3]),
           lambda: unsort_tokens(rows, o, w.bfloat16()), lambda: unsort_tokens(rows, o, w, residual=x[:, :8]),
           lambda: sort_tokens(x, o, scale=w.half()), lambda: sort_tokens(x[:, :0], o),
           lambda: sort_tokens(x, TokenOrder(o.row_of.long(), o.route_of, o.offsets)),
           lambda: sort_tokens(x, TokenOrder(o.row_of, o.route_of[:-1], o.offsets)),
           lambda: sort_tokens(x, TokenOrder(o.row_of.cpu(), o.route_of, o.offsets)),
           lambda: sort_tokens(x.float().requires_grad_(), o, scale=w),
           lambda: sort_routes(idx[:1, :1].expand(2 ** 32 + 1, 1), E)]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    for f in (lambda: sort_routes(idx.float(), E), lambda: sort_routes(idx[0], E), lambda: sort_tokens(x.long(), o),
              lambda: unsort_tokens(rows.to(torch.float8_e4m3fn), o, w), lambda: sort_tokens(x.cpu(), o),
              lambda: unsort_tokens(rows, o, w, out_dtype=torch.float64)):
        with pytest.raises(TypeError):
            f()
    for n, first in ((0, 0), (1025, 0), (E, -1), (E, 2 ** 32)):
        with pytest.raises(ValueError):
            sort_routes(idx, n, first_expert=first)


@gpu
def test_an_order_out_of_range_touches_nothing():
    """Row numbers outside the rows are skipped by the kernels' own checks, rows in use are clamped."""
    from constellation_b200.token_sort import TokenOrder, sort_tokens, unsort_tokens, unsort_tokens_backward

    T, K, H = 3, 2, 64
    row_of = torch.tensor([[0, 99], [-5, 2 ** 31 - 1], [6, 1]], dtype=torch.int32, device="cuda")
    o = TokenOrder(row_of, torch.zeros(6, dtype=torch.int32, device="cuda"),
                   torch.tensor([0, 1 << 30], dtype=torch.int32, device="cuda"))
    x, rows, w = rand((T, H), torch.float32, 1), rand((6, H), torch.float32, 2), torch.ones(T, K, device="cuda")
    assert torch.equal(sort_tokens(x, o)[:2], x[[0, 2]])
    out = unsort_tokens(rows, o, w)
    assert torch.equal(out[0], rows[0]) and (out[1] == 0).all() and torch.equal(out[2], rows[1])
    d_rows, d_w = unsort_tokens_backward(x, rows, o, w)
    assert torch.equal(d_rows[:2], x[[0, 2]]) and (d_w[[0, 1, 1, 2], [1, 0, 1, 0]] == 0).all()


def test_refusals_without_a_device(monkeypatch):
    from constellation_b200 import _lib, token_sort
    from constellation_b200.token_sort import TokenOrder, sort_routes, sort_tokens, unsort_tokens

    idx = torch.zeros(2, 2, dtype=torch.int32)
    o = TokenOrder(idx, idx.view(-1), torch.zeros(3, dtype=torch.int32))
    for f in (lambda: sort_routes(idx, 4), lambda: sort_tokens(torch.zeros(2, 8), o),
              lambda: unsort_tokens(torch.zeros(4, 8), o)):
        with pytest.raises(TypeError):
            f()
    L, P, BAD = _lib.lib, 16, _lib.CST_ERR_INVALID_ARG
    for a in ((P, 2, 1, 1, 4, 0), (P, 4, -1, 1, 4, 0), (P, 4, 1, 0, 4, 0), (P, 4, 1, 1025, 4, 0),
              (P, 4, 1, 1, 0, 0), (P, 4, 1, 1, 1025, 0), (P, 4, 1, 1, 4, -1), (None, 4, 1, 1, 4, 0),
              (P, 4, 2 ** 30, 2, 4, 0)):
        assert L.cst_sort_routes(*a, P, P, P, None) == BAD, a
    assert L.cst_sort_routes(P, 4, 1, 1, 4, 0, P, P, None, None) == BAD
    rows = lambda x=P, n=64, ld=64, s=None, ns=0, lds=0, T=1, K=1, out=P: L.cst_sort_rows(  # noqa: E731
        x, n, ld, s, ns, lds, T, K, P, P, out, None, None)
    assert rows(x=None, T=0, out=None) == _lib.CST_OK
    for kw in (dict(n=0), dict(ld=63), dict(s=P, ns=0), dict(s=P, ns=4, lds=3), dict(T=-1), dict(K=0), dict(x=None),
               dict(out=None), dict(s=P, ns=1, lds=1)):
        assert rows(**kw) == BAD, kw
    un = lambda r=P, dt=2, ld=64, T=1, K=1, H=64, res=None, rt=2, ldr=64, out=P, ot=2: L.cst_unsort_rows(  # noqa: E731
        r, dt, ld, P, None, T, K, H, res, rt, ldr, out, ot, None)
    assert un(r=None, T=0, out=None) == _lib.CST_OK
    for kw in (dict(dt=4), dict(ot=0), dict(res=P, rt=9), dict(ld=63), dict(H=0), dict(H=2 ** 30 + 1, ld=2 ** 40),
               dict(res=P, ldr=1), dict(r=None), dict(out=None), dict(K=2000)):
        assert un(**kw) == BAD, kw
    gr = lambda g=P, gt=2, ldg=64, r=P, dt=2, ld=64, T=1, H=64, dr=P, dw=P: L.cst_unsort_rows_grad(  # noqa: E731
        g, gt, ldg, r, dt, ld, P, P, P, T, 1, H, dr, dw, None)
    assert gr(g=None, T=0) == _lib.CST_OK and gr(dr=None, dw=None) == _lib.CST_OK
    for kw in (dict(gt=4), dict(dt=0), dict(ldg=1), dict(ld=1), dict(H=0), dict(g=None), dict(r=None)):
        assert gr(**kw) == BAD, kw
    # autograd under capture is refused before anything is launched
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        token_sort._refuse_capture("sort_tokens")
