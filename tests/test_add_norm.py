"""Residual add + RMSNorm, to 16 or 32 bits and to e4m3 with scales, against the formula in 64 bits.

Bounds: a result is one rounding of an fp32 chain.  The chain's relative error is that of the sum
of squares (at most 32 + 5 + 32 sequential additions of positive terms, halved by the root), the root (2 units),
and 3 products: below 48 * 2^-24.  A rounding to type t adds eps(t) / 2 of the value, or half its
smallest step.  e4m3: 2^-4 of the value, or half the subnormal step, 2^-10, times the scale.
"""
import math

import pytest
import torch

REL = 48 * 2.0 ** -24
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def tiny(dt):
    return {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}[dt]


def close(got, ref, dt):
    bound = ref.abs() * (torch.finfo(dt).eps / 2 + REL) + tiny(dt)
    assert ((got.double() - ref).abs() <= bound).all(), ((got.double() - ref).abs() - bound).max()


def formula(x, res, w, eps=1e-6):
    h = x.double() + (res.double() if res is not None else 0)
    y = h / (h.square().mean(1, keepdim=True) + eps).sqrt()
    return h, y if w is None else y * w.double()


def make(T, H, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(T, H, generator=g) * 2).to("cuda", dt), torch.randn(T, H, generator=g).to("cuda", dt),
            (1 + 0.1 * torch.randn(H, generator=g)).cuda())


def check8(q, scale, y):
    T, H = y.shape
    B = (H + 127) // 128
    assert q.dtype == torch.float8_e4m3fn and q.shape == (T, H) and scale.shape == (T, B)
    for b in range(B):
        part, s = y[:, b * 128:(b + 1) * 128], scale[:, b].double()
        most = part.abs().amax(1)
        want = torch.where(most > 0, most / 448, torch.ones_like(most))
        assert ((s - want).abs() <= want * (REL + 2.0 ** -23)).all()
        back = q[:, b * 128:(b + 1) * 128].double() * s[:, None]
        assert ((back - part).abs() <= part.abs() * (2.0 ** -4 + REL) + 2.0 ** -10 * s[:, None] * (1 + REL)).all()


WIDTHS = [1, 2, 7, 8, 64, 127, 128, 136, 1000, 1024, 1025, 5001, 7168, 8192, 8200, 16384, 32767, 32768]


@gpu
@pytest.mark.parametrize("H", WIDTHS)
@pytest.mark.parametrize("T", [1, 5])
def test_widths(T, H):
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    x, res, w = make(T, H, torch.bfloat16, H)
    h, y = formula(x, res, w)
    out, s = add_rms_norm(x, res, w)
    close(out, y, torch.bfloat16)
    close(s, h, torch.bfloat16)
    q, scale, s8 = add_rms_norm_fp8(x, res, w)
    check8(q, scale, y)
    assert torch.equal(s8, s)


@gpu
@pytest.mark.parametrize("H", [250, 256, 7168])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rt", DTYPES)
def test_types(H, dt, rt):
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    x, _, w = make(33, H, dt)
    _, res, _ = make(33, H, rt, 1)
    h, y = formula(x, res, w)
    out, s = add_rms_norm(x, res, w)
    assert out.dtype == dt and s.dtype == rt
    close(out, y, dt)
    close(s, h, rt)
    out32 = torch.empty(33, H, device="cuda")
    add_rms_norm(x, res, w, out=out32)
    close(out32, y, torch.float32)
    q, scale, s8 = add_rms_norm_fp8(x, res, w)
    check8(q, scale, y)
    assert torch.equal(s8, s)
    _, y0 = formula(x, None, None)
    q, scale, none = add_rms_norm_fp8(x)
    assert none is None
    check8(q, scale, y0)


@gpu
@pytest.mark.parametrize("T", [1, 147, 148, 149, 600, 4096])
def test_batches_agree_with_single_rows(T):
    """A row's result does not depend on the batch it is in."""
    from constellation_b200.context import add_rms_norm_fp8

    x, res, w = make(T, 1536, torch.bfloat16, T)
    q, scale, s = add_rms_norm_fp8(x, res, w)
    check8(q, scale, formula(x, res, w)[1])
    for t in (0, T // 2, T - 1):
        one = add_rms_norm_fp8(x[t:t + 1], res[t:t + 1], w)
        check8(one[0], one[1], formula(x[t:t + 1], res[t:t + 1], w)[1])
        assert torch.equal(one[2], s[t:t + 1])


@gpu
@pytest.mark.parametrize("H,offset,stride", [(256, 0, 264), (256, 3, 300), (255, 1, 257), (7168, 8, 7200)])
def test_strides_and_offsets(H, offset, stride):
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    g = torch.Generator().manual_seed(3)
    wide = torch.randn(9, stride + 8, generator=g).to("cuda", torch.float16)
    x = wide[:, offset:offset + H]
    res = torch.randn(H, 9, generator=g).to("cuda", torch.float16).t()  # columns apart: copied
    h, y = formula(x, res, None)
    room = torch.full((9, stride), 7.0, device="cuda", dtype=torch.float16)
    sums = torch.full((9, stride + 1), 7.0, device="cuda", dtype=torch.float16)
    out, s = add_rms_norm(x, res, out=room[:, :H], sum_out=sums[:, 1:H + 1])
    close(out, y, torch.float16)
    close(s, h, torch.float16)
    assert (room[:, H:] == 7).all() and (sums[:, 0] == 7).all() and (sums[:, H + 1:] == 7).all()
    q, scale, _ = add_rms_norm_fp8(x, res)
    check8(q, scale, y)


@gpu
@pytest.mark.parametrize("T,H,offset,stride", [(640, 8, 0, 8), (640, 250, 0, 256), (700, 256, 8, 272), (1300, 2048, 0, 2048),
                                               (640, 8192, 0, 8192), (640, 5001, 1, 5003), (3, 9001, 1, 9003),
                                               (640, 9001, 0, 9001), (700, 8200, 0, 8200), (301, 16384, 8, 16400)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_many_rows(T, H, offset, stride, dt):
    """Long batches go from row to row: a row's numbers reach no other row, with and without what is optional."""
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    g = torch.Generator().manual_seed(H)
    x = (torch.randn(T, stride + 8, generator=g) * 2).to("cuda", dt)[:, offset:offset + H]
    res = torch.randn(T, stride + 8, generator=g).to("cuda", dt)[:, offset:offset + H]
    w = (1 + 0.1 * torch.randn(H, generator=g)).cuda()
    h, y = formula(x, res, w)
    room = torch.full((T, stride + 8), 7.0, device="cuda", dtype=dt)
    out, s = add_rms_norm(x, res, w, out=room[:, offset:offset + H])
    close(out, y, dt)
    close(s, h, dt)
    assert (room[:, :offset] == 7).all() and (room[:, offset + H:] == 7).all()
    q, scale, s8 = add_rms_norm_fp8(x, res, w)
    check8(q, scale, y)
    assert torch.equal(s8, s)
    bad = x.clone()
    bad[T // 2] = math.nan
    keep = torch.arange(T, device="cuda") != T // 2
    q1, scale1, _ = add_rms_norm_fp8(bad, res, w)
    assert torch.equal(q1.view(torch.uint8)[keep], q.view(torch.uint8)[keep]) and torch.equal(scale1[keep], scale[keep])
    _, y0 = formula(x, None, None)
    q, scale, none = add_rms_norm_fp8(x)
    assert none is None
    check8(q, scale, y0)


@gpu
def test_in_place():
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    x, res, w = make(40, 7168, torch.bfloat16)
    out, s = add_rms_norm(x, res, w)
    q, scale, _ = add_rms_norm_fp8(x, res, w)
    r = res.clone()
    out2, s2 = add_rms_norm(x, r, w, sum_out=r)
    assert s2.data_ptr() == r.data_ptr() and torch.equal(r, s) and torch.equal(out2, out)
    x2, r = x.clone(), res.clone()
    add_rms_norm(x2, r, w, out=x2, sum_out=r)
    assert torch.equal(x2, out) and torch.equal(r, s)
    x2 = x.clone()
    q2, scale2, _ = add_rms_norm_fp8(x2, res, w, sum_out=x2)
    assert torch.equal(x2, s) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scale2, scale)


@gpu
@pytest.mark.parametrize("H", [256, 255])
def test_zero_tiny_and_huge_rows(H):
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    x = torch.zeros(6, H, device="cuda")
    x[1] = 1e-18                      # squares far below the smallest normal: eps decides
    x[2, :128] = 1.0                  # one block of values beside blocks of zeros
    x[3] = 3e4
    x[4, 5] = 1e-38                   # a block whose scale would be subnormal
    x[5] = -2.0
    res = torch.zeros_like(x)
    h, y = formula(x, res, None)
    out, s = add_rms_norm(x, res)
    assert torch.equal(s, x)
    close(out[[0, 2, 3, 5]], y[[0, 2, 3, 5]], torch.float32)
    q, scale, _ = add_rms_norm_fp8(x)
    check8(q[[0, 1, 2, 3, 5]], scale[[0, 1, 2, 3, 5]], y[[0, 1, 2, 3, 5]])
    assert (scale[0] == 1).all() and (q[0].float() == 0).all() and (scale[2, 1:] == 1).all()
    assert torch.isfinite(scale).all() and torch.isfinite(q.float()).all()


@gpu
@pytest.mark.parametrize("H", [256, 301])
def test_infinities_and_nan_stay_in_their_rows(H):
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    x, res, w = make(4, H, torch.float32)
    clean = add_rms_norm(x, res, w)[0]
    x[1, 3], x[2, 200] = math.nan, math.inf
    out, _ = add_rms_norm(x, res, w)
    assert torch.equal(out[[0, 3]], clean[[0, 3]])
    assert torch.isnan(out[1]).all()          # the row's mean is NaN
    assert torch.isnan(out[2, 200]) and (out[2, :200] == 0).all() and (out[2, 201:] == 0).all()
    q, scale, _ = add_rms_norm_fp8(x, res, w)
    assert torch.isnan(q[1].float()).all() and torch.isnan(q[2, 200].float())
    assert (scale[2] == 1).all() and (q[2, :200].float() == 0).all()
    check8(q[[0, 3]], scale[[0, 3]], formula(x[[0, 3]], res[[0, 3]], w)[1])


@gpu
def test_empty_batch_side_stream_and_graph():
    from constellation_b200.context import add_rms_norm_fp8

    x, res, w = make(64, 7168, torch.bfloat16)
    q, scale, s = add_rms_norm_fp8(x[:0], res[:0], w)
    assert q.shape == (0, 7168) and scale.shape == (0, 56) and s.shape == (0, 7168)
    want = add_rms_norm_fp8(x, res, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = add_rms_norm_fp8(x, res, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = add_rms_norm_fp8(x, res, w)
    x.copy_(x.flip(0))
    res.copy_(res.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0].view(torch.uint8), want[0].view(torch.uint8).flip(0))
    assert torch.equal(held[1], want[1].flip(0)) and torch.equal(held[2], want[2].flip(0))


@gpu
def test_refusals_of_device_tensors():
    from constellation_b200 import _lib
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    x, res, w = make(4, 256, torch.bfloat16)
    bad = [lambda: add_rms_norm(x, res[:3], w), lambda: add_rms_norm(x, res, w[:255]),
           lambda: add_rms_norm(x, res, w.bfloat16()), lambda: add_rms_norm(x, res.cpu(), w),
           lambda: add_rms_norm(x, res, w, sum_out=torch.empty(4, 256, device="cuda")),
           lambda: add_rms_norm(x, res, w, out=torch.empty(256, 4, device="cuda").t()),
           lambda: add_rms_norm(x, res, w, out=torch.empty(1, 256, device="cuda").expand(4, 256)),
           lambda: add_rms_norm_fp8(x, None, w, sum_out=res), lambda: add_rms_norm(x.float().requires_grad_(), res, w),
           lambda: add_rms_norm_fp8(x[:1, :1].expand(2 ** 32 + 1, 1))]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    for f in (lambda: add_rms_norm(x, None, w), lambda: add_rms_norm(x.double(), res, w),
              lambda: add_rms_norm(x[0], res, w), lambda: add_rms_norm(x, res.double(), w)):
        with pytest.raises(TypeError):
            f()
    wide = torch.zeros(1, 32769, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(_lib.CstError):
        add_rms_norm_fp8(wide)


def test_refusals_without_a_device():
    from constellation_b200 import _lib
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    x = torch.zeros(2, 8)
    for f in (lambda: add_rms_norm(x, x), lambda: add_rms_norm_fp8(x), lambda: add_rms_norm_fp8(None)):
        with pytest.raises(TypeError):
            f()
    L, P = _lib.lib, 16

    def call(x=P, xt=2, ldx=256, res=P, rt=2, ldr=256, T=1, H=256, sum_=None, lds=256, out=P, ot=2, ldo=256,
             scale=None):
        return L.cst_add_rmsnorm(x, xt, ldx, res, rt, ldr, T, H, None, 1e-6, sum_, lds, out, ot, ldo, scale, None)

    assert call(x=None, res=None, out=None, T=0) == _lib.CST_OK
    for kw in (dict(xt=4), dict(rt=0), dict(ot=5), dict(H=0), dict(H=32769), dict(T=-1), dict(T=2 ** 30 + 1), dict(ldx=255), dict(ldr=1),
               dict(ldo=255), dict(sum_=P, lds=8), dict(x=None), dict(out=None), dict(ot=4), dict(res=None, sum_=P)):
        assert call(**kw) == _lib.CST_ERR_INVALID_ARG, kw
        assert _lib.last_error()
