"""The operators around the layer have no forward-mode derivatives: a tangent is refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

gpu = pytest.mark.gpu


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def test_a_tangent_is_seen():
    from constellation_b200.context import _no_grad, _no_tangent

    x = torch.ones(3)
    _no_tangent("it", x, None)
    with forward_ad.dual_level():
        d = dual(x)
        for refuse in (_no_tangent, _no_grad):
            refuse("it", x, None, d.detach())
            for mode in (torch.no_grad, torch.enable_grad):
                with mode(), pytest.raises(RuntimeError, match="it has no forward-mode derivative"):
                    refuse("it", None, x, d)
    _no_tangent("it", x)


def calls():
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8
    from constellation_b200.int4 import Int4Weight, grouped_int4, quantize_int4
    from constellation_b200.token_sort import (sort_routes, sort_tokens, sort_tokens_backward, unsort_tokens,
                                               unsort_tokens_backward)

    g = torch.Generator().manual_seed(1)
    x, residual, grad = (torch.randn(6, 128, generator=g).cuda() for _ in range(3))
    weight, w = torch.rand(128, generator=g).cuda(), torch.rand(6, 2, generator=g).cuda()
    order = sort_routes(torch.randint(0, 4, (6, 2), generator=g).cuda(), 4)
    rows = sort_tokens(x, order)
    half = x.to(torch.bfloat16)
    q, s, _ = quantize_int4(torch.randn(16, 128, generator=g).cuda())
    held = Int4Weight(q, s)
    return [(add_rms_norm, (x, residual, weight)), (add_rms_norm_fp8, (x, residual, weight)), (grouped_int4, (half, held)),
            (sort_tokens, (x, order)), (lambda x, s: sort_tokens(x, order, scale=s), (x, x[:, :1].contiguous())),
            (unsort_tokens, (rows, order, w)), (lambda r, e: unsort_tokens(r, order, residual=e), (rows, residual)),
            (sort_tokens_backward, (rows, order)), (unsort_tokens_backward, (grad, rows, order, w)),
            (lambda q, s: Int4Weight(q, s), (q, s))]


@gpu
@pytest.mark.parametrize("at", range(10))
def test_a_tangent_is_refused(at):
    f, args = calls()[at]
    f(*args)
    for i, t in enumerate(args):
        if not isinstance(t, torch.Tensor) or not t.is_floating_point():
            continue
        with forward_ad.dual_level():
            d = dual(t)
            f(*args)  # others' tangents do not matter
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                f(*args[:i], d, *args[i + 1:])
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                f(*args[:i], d, *args[i + 1:])


@gpu
def test_a_tangent_of_a_gradient_is_refused():
    from constellation_b200.token_sort import sort_routes, sort_tokens, unsort_tokens

    x = torch.randn(6, 128, device="cuda", requires_grad=True)
    order = sort_routes(torch.zeros(6, 2, dtype=torch.int64, device="cuda"), 2)
    rows = sort_tokens(x, order)
    out = unsort_tokens(rows, order, torch.ones(6, 2, device="cuda"))
    for y, of in ((rows, x), (out, rows)):
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(y, (of,), dual(torch.ones_like(y)), retain_graph=True)
        torch.autograd.grad(y, (of,), torch.ones_like(y), retain_graph=True)
