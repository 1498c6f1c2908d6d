"""Grouped products with 4-bit weights and the layer over them, against the definitions in 64 bits.

Bound of a product.  The products q x and zero x are exact in fp32 and each 32 k of both are added up before
the next, so the error is that of the sums: at most one unit of 2^-23 of the sum of magnitudes for each of
`group` additions inside a group (the matrix units need not round to nearest), then two roundings a
group and a tree over parts of k: (group + 2 K / group + 64) * 2^-23 of sum |W x|.  Where zero points leave
little of a group, its magnitude is that of scale (q + zero) |x|, and `check` is given those weights as `mag`.
x itself is kept exactly down to 2^-13 (bf16) or 2^-11 (fp16) of its row's largest; what a smaller one loses
is below 2^-21 (2^-22) of that largest, `drop`, which counts where a row has outliers: rows of randn hold no |x|
above 6, so that drop * 6 * sum |W| is below 2^-18 sum |W|, a hundredth of the first term for their mean |x| of 0.8.
The result is rounded once, eps(t) / 2 of the value.  silu has a slope below 1.1 and costs 8 * 2^-24 of its
value.
"""
import math

import pytest
import torch

gpu = pytest.mark.gpu
U = 2.0 ** -23


def make_weight(E, N, K, group, zeros, scale_dtype=torch.float16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 16, (E, N, K), generator=g, device="cuda", dtype=torch.uint8)
    scale = (torch.rand(E, N, K // group, generator=g, device="cuda") * 0.02 + 0.002).to(scale_dtype)
    zero = torch.randint(0, 16, (E, N, K // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    z = 8.0 if zero is None else zero.double().repeat_interleave(group, 2)
    return q[..., 0::2] | (q[..., 1::2] << 4), scale, zero, \
        (q.double() - z) * scale.double().repeat_interleave(group, 2)


def make_x(R, K, dt, seed=1):
    x = torch.randn(R, K, generator=torch.Generator().manual_seed(seed)).cuda()
    if dt != torch.float8_e4m3fn:
        return x.to(dt), None, x.to(dt).double()
    q = (x * 100).clamp(-448, 448).to(dt)
    s = torch.rand(R, (K + 127) // 128, generator=torch.Generator().manual_seed(seed + 1)).cuda() + 0.5
    return q, s, q.double() * s.double().repeat_interleave(128, 1)[:, :K]


def check(out, x64, W, offsets, group, swiglu, mag=None, drop=0.0):
    """Every row of every expert against W[e] x in 64 bits; the others are zero."""
    sizes = W.abs() if mag is None else mag
    K, N = W.shape[2], W.shape[1]
    at = offsets.tolist() if offsets is not None else [0, x64.shape[0]]
    g = (group + 2 * K / group + 64) * U
    end = torch.finfo(out.dtype)
    seen = torch.zeros(x64.shape[0], dtype=torch.bool)
    for e in range(W.shape[0]):
        lo, hi = at[e], at[e + 1]
        seen[lo:hi] = True
        y, most = x64[lo:hi] @ W[e].T, x64[lo:hi].abs().amax(1, keepdim=True) if hi > lo else 0.0
        err = g * (x64[lo:hi].abs() @ sizes[e].T) + drop * most * W[e].abs().sum(1)
        if swiglu:
            u, v, du, dv = y[:, :N // 2], y[:, N // 2:], err[:, :N // 2], err[:, N // 2:]
            s = v * torch.sigmoid(v)
            y, err = s * u, s.abs() * du + 1.1 * u.abs() * dv + 1.1 * du * dv + 8 * 2.0 ** -24 * (s * u).abs()
        bound = err + y.abs() * end.eps / 2 + end.smallest_normal
        got = out[lo:hi].double()
        assert ((got - y).abs() <= bound).all(), (e, ((got - y).abs() / bound).max())
    assert (out[~seen.cuda()] == 0).all()


def offsets_of(counts):
    return torch.tensor([0] + list(counts), device="cuda").cumsum(0).to(torch.int32)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N,K", [(64, 128), (1, 128), (63, 384), (200, 896), (129, 2048)])
def test_products(N, K, zeros, group, dt):
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(3, N, K, group, zeros)
    w = Int4Weight(q, s, z)
    off = offsets_of((2, 0, 5))
    x, xs, x64 = make_x(9, K, dt)
    out = grouped_int4(x, w, off, x_scale=xs)
    assert out.shape == (9, N) and out.dtype == (torch.bfloat16 if xs is not None else dt)
    check(out, x64, W, off, group, False)
    check(grouped_int4(x, w, off, x_scale=xs, out_dtype=torch.float32), x64, W, off, group, False)


@gpu
@pytest.mark.parametrize("R", [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 64, 65, 130])
def test_row_counts(R):
    from constellation_b200.int4 import Int4Weight, grouped_int4

    N, K = 192, 640
    q, s, z, W = make_weight(1, N, K, 128, True)
    w = Int4Weight(q[0], s[0], z[0])
    x, _, x64 = make_x(R, K, torch.bfloat16)
    out = grouped_int4(x, w)
    assert out.shape == (R, N)
    check(out, x64, W, None, 128, False)
    off = torch.tensor([0, R], dtype=torch.int32, device="cuda")
    assert torch.equal(grouped_int4(x, w, off), out)


@gpu
@pytest.mark.parametrize("counts", [(0, 0, 0, 0), (1, 1, 1, 1), (0, 0, 0, 40), (70, 0, 3, 0), (33, 16, 9, 8),
                                    (1, 200, 1, 0)])
@pytest.mark.parametrize("tail", [0, 5])
def test_ragged_experts(counts, tail):
    from constellation_b200.int4 import Int4Weight, grouped_int4

    N, K = 320, 1152
    q, s, z, W = make_weight(4, N, K, 64, False, torch.bfloat16)
    w = Int4Weight(q, s)
    off = offsets_of(counts)
    R = sum(counts) + tail
    x, _, x64 = make_x(R, K, torch.float16)
    x[sum(counts):] = math.nan  # rows of no expert are not used
    check(grouped_int4(x, w, off), x64, W, off, 64, False)
    if R:
        lead = torch.cat([off[:1] + 1, (off[1:] + 1).clamp(max=R)]).to(torch.int32)  # a row before the first expert
        x, _, x64 = make_x(R, K, torch.float16)
        check(grouped_int4(x, w, lead), x64, W, lead, 64, False)


@gpu
@pytest.mark.parametrize("I", [1, 16, 31, 32, 33, 200])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float8_e4m3fn])
def test_swiglu(I, dt):
    from constellation_b200.int4 import Int4Weight, grouped_int4

    K = 512
    q, s, z, W = make_weight(2, 2 * I, K, 128, True, torch.float32)
    w = Int4Weight(q, s, z, swiglu=True)
    off = offsets_of((3, 11))
    x, xs, x64 = make_x(14, K, dt)
    for od in (torch.float32, torch.bfloat16, torch.float16):
        out = grouped_int4(x / 8 if xs is None else x, w, off, x_scale=None if xs is None else xs / 800, out_dtype=od)
        assert out.shape == (14, I)
        check(out, (x / 8).double() if xs is None else x.double() * (xs / 800).double().repeat_interleave(128, 1), W,
              off, 128, True)


@gpu
@pytest.mark.parametrize("E,N,K,R", [(1, 4096, 7168, 1), (1, 7168, 2048, 3), (1, 64, 16384, 2), (8, 1024, 2048, 64),
                                     (300, 64, 256, 500), (1024, 64, 128, 700), (2, 2048, 1024, 600)])
def test_larger_shapes(E, N, K, R):
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(E, N, K, 128, False)
    w = Int4Weight(q, s)
    g = torch.Generator().manual_seed(E)
    counts = torch.bincount(torch.randint(0, E, (R,), generator=g), minlength=E).tolist()
    off = offsets_of(counts)
    x, _, x64 = make_x(R, K, torch.bfloat16)
    out = grouped_int4(x, w, off)
    check(out, x64, W, off, 128, False)
    assert torch.equal(grouped_int4(x, w, off), out)  # repeats bit for bit


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("K,width,offset", [(96, 131, 1), (160, 168, 0), (352, 360, 8), (1056, 1057, 0)])
def test_strided_rows_and_what_lies_behind_them(K, width, offset, dt):
    """Columns past k belong to someone else: NaN there must not reach a result."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(1, 96, K, 32, True)
    w = Int4Weight(q, s, z)
    x, xs, x64 = make_x(11, K, dt)
    wide = torch.full((11, width + 8), math.nan, device="cuda").to(dt)
    wide[:, offset:offset + K] = x
    got = grouped_int4(wide[:, offset:offset + K], w, x_scale=xs)
    check(got, x64, W, None, 32, False)
    assert torch.equal(grouped_int4(x, w, x_scale=xs), got)
    if xs is not None:
        room = torch.full((11, xs.shape[1] + 3), math.nan, device="cuda")
        room[:, 2:2 + xs.shape[1]] = xs
        assert torch.equal(grouped_int4(x, w, x_scale=room[:, 2:2 + xs.shape[1]]), got)


@gpu
def test_infinities_and_nan_stay_in_their_rows():
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(2, 128, 256, 128, False)
    w, off = Int4Weight(q, s), offsets_of((9, 9))
    x, _, _ = make_x(18, 256, torch.bfloat16)
    clean = grouped_int4(x, w, off)
    x[3, 7], x[12, 0] = math.nan, math.inf
    out = grouped_int4(x, w, off)
    keep = [r for r in range(18) if r not in (3, 12)]
    assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[3]).all()
    assert not torch.isfinite(out[12]).any()


@gpu
@pytest.mark.parametrize("R", [3, 12, 40, 75])
@pytest.mark.parametrize("chunks", [1, 2, 3, 4, 5, 9])
@pytest.mark.parametrize("group,zeros", [(128, False), (64, True), (32, True)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
def test_tiles_and_part_steps(R, chunks, group, zeros, dt):
    """Every tile of rows, steps that end inside a step's chunks, k split over CTAs or not, and the last chunk part."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    K = 128 * chunks - (32 if group == 32 else 0)
    q, s, z, W = make_weight(2, 144, K, group, zeros, seed=chunks)
    w = Int4Weight(q, s, z)
    off = offsets_of((R, R // 3))
    x, xs, x64 = make_x(R + R // 3, K, dt, R)
    out = grouped_int4(x, w, off, x_scale=xs, out_dtype=torch.float32)
    check(out, x64, W, off, group, False)
    assert torch.equal(grouped_int4(x, w, off, x_scale=xs, out_dtype=torch.float32), out)


@gpu
@pytest.mark.parametrize("dt,drop", [(torch.bfloat16, 2.0 ** -21), (torch.float16, 2.0 ** -22)])
@pytest.mark.parametrize("factor", [16.0, 1000.0, 10000.0])
def test_outliers_in_a_row(factor, dt, drop):
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(1, 136, 1152, 128, False)
    x, _, _ = make_x(20, 1152, torch.float32)
    x[torch.arange(20), torch.arange(20) * 57] *= factor
    x[7] *= 2.0 ** -12
    x[8] = 0
    x = x.to(dt)
    out = grouped_int4(x, Int4Weight(q, s, z), out_dtype=torch.float32)
    check(out, x.double(), W, None, 128, False, drop=drop)
    assert (out[8] == 0).all()


@gpu
@pytest.mark.parametrize("dt,lo,hi", [(torch.bfloat16, -30, 30), (torch.float16, -10, 8)])
def test_numbers_of_every_size(dt, lo, hi):
    """Rows from the smallest to the largest of the type."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(1, 64, 256, 64, True)
    x, _, _ = make_x(hi - lo, 256, torch.float32)
    x = (x * torch.exp2(torch.arange(lo, hi, device="cuda").float())[:, None]).to(dt)
    out = grouped_int4(x, Int4Weight(q, s, z), out_dtype=torch.float32)
    check(out, x.double(), W, None, 64, False, drop=2.0 ** -21)


@gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
def test_weights_at_their_zero_point(zeros, dt):
    """Groups of nothing but zero points: what is left is the rounding of sums that cancel."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    N, K, G = 64, 512, 64
    g = torch.Generator().manual_seed(5)
    zero = torch.randint(0, 16, (1, N, K // G), generator=g, dtype=torch.uint8) if zeros else \
        torch.full((1, N, K // G), 8, dtype=torch.uint8)
    v = zero.repeat_interleave(G, 2)
    v[:, :, 7] = (v[:, :, 7] + 1) % 16
    scale = torch.rand(1, N, K // G, generator=g) + 0.5
    q, zero, scale = (v[..., 0::2] | (v[..., 1::2] << 4)).cuda(), zero.cuda(), scale.cuda()
    z64, s64 = (t.double().repeat_interleave(G, 2) for t in (zero, scale))
    w = Int4Weight(q, scale, zero if zeros else None)
    x, xs, x64 = make_x(5, K, dt)
    out = grouped_int4(x, w, x_scale=xs, out_dtype=torch.float32)
    check(out, x64, (v.cuda().double() - z64) * s64, None, G, False, mag=(v.cuda().double() + z64) * s64)


@gpu
def test_two_products_at_once():
    """One weight, two streams at the same time, each call with its own workspace."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(8, 1024, 1024, 128, False)
    w, off = Int4Weight(q, s), offsets_of((5, 0, 9, 1, 1, 17, 2, 3))
    xs = [make_x(38, 1024, dt, i)[0] for i, dt in enumerate((torch.bfloat16, torch.float16))]
    want = [grouped_int4(x, w, off) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(10):
        for i, x in enumerate(xs):
            with torch.cuda.stream(streams[i]):
                got[i].append(grouped_int4(x, w, off))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
    w.device_error()


@gpu
def test_out_streams_and_graphs():
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(4, 256, 512, 128, False)
    w, off = Int4Weight(q, s), offsets_of((3, 0, 20, 1))
    x, _, _ = make_x(26, 512, torch.bfloat16)
    want = grouped_int4(x, w, off)
    room = torch.full((26, 256), 3.0, device="cuda", dtype=torch.bfloat16)
    assert grouped_int4(x, w, off, out=room) is room and torch.equal(room, want) and (room[24:] == 0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grouped_int4(x, w, off)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(grouped_int4(x, w, off))
    off.copy_(offsets_of((0, 24, 0, 2)))
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], held[1]) and torch.equal(held[0], grouped_int4(x, w, off))


@gpu
def test_offsets_out_of_order_stay_in_range():
    """Offsets that are no offsets give unspecified rows and touch nothing outside x and out."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(3, 64, 128, 128, False)
    w = Int4Weight(q, s)
    x, _, x64 = make_x(10, 128, torch.bfloat16)
    room = torch.full((30, 64), 5.0, device="cuda", dtype=torch.bfloat16)
    for off in ([-7, 4, 1 << 30, 9], [9, 3, 0, 0], [0, 0, 0, -5], [1 << 30] * 4):
        grouped_int4(x, w, torch.tensor(off, dtype=torch.int32, device="cuda"), out=room[10:20])
        torch.cuda.synchronize()
        assert (room[:10] == 5).all() and (room[20:] == 5).all()


@gpu
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 128])
def test_quantiser(group, symmetric):
    from constellation_b200.int4 import Int4Weight, grouped_int4, quantize_int4

    g = torch.Generator().manual_seed(2)
    w = torch.randn(80, 256, generator=g).cuda() * 0.02 + (0 if symmetric else 0.01)
    w[3, :group] = 0
    q, s, z = quantize_int4(w, group, symmetric=symmetric)
    back = torch.stack((q & 15, q >> 4), -1).view(80, 256).double()
    back = (back - (8.0 if z is None else z.double().repeat_interleave(group, 1))) \
        * s.double().repeat_interleave(group, 1)
    step = s.double().repeat_interleave(group, 1)
    # half a step; at the ends of the range the stored scale's rounding (2^-11 of at most 15 steps), and
    # with zero points half a step more, since the zero point is rounded too
    assert ((back - w.double()).abs() <= step * (0.5 + 15 * 2.0 ** -11 + (0 if symmetric else 0.5))).all()
    assert (back[3, :group] == 0).all()
    x, _, x64 = make_x(3, 256, torch.bfloat16)
    check(grouped_int4(x, Int4Weight(q, s, z)), x64, back[None], None, group, False)


@gpu
def test_the_operators_together():
    """Norm to 8 bits, sort, both products, back with weights, against the chain in 64 bits."""
    from constellation_b200.context import add_rms_norm_fp8
    from constellation_b200.int4 import Int4Weight, grouped_int4
    from constellation_b200.token_sort import sort_routes, sort_tokens, unsort_tokens

    T, K, E, H, I = 23, 3, 5, 640, 96
    qu, su, zu, Wu = make_weight(E, 2 * I, H, 64, True, seed=1)
    qd, sd, zd, Wd = make_weight(E, H, I, 32, False, seed=2)
    up, down = Int4Weight(qu, su, zu, swiglu=True), Int4Weight(qd, sd)
    g = torch.Generator().manual_seed(4)
    x, res = (torch.randn(T, H, generator=g).to("cuda", torch.bfloat16) for _ in range(2))
    idx = torch.randint(-1, E, (T, K), generator=g).cuda()
    weight = torch.rand(T, K, generator=g).cuda()
    q8, s8, h = add_rms_norm_fp8(x, res)
    order = sort_routes(idx, E)
    rows, rs = sort_tokens(q8, order, scale=s8)
    mid = grouped_int4(rows, up, order.offsets, x_scale=rs)
    y = grouped_int4(mid, down, order.offsets, out_dtype=torch.float32)
    out = unsort_tokens(y, order, weight, residual=h, out_dtype=torch.float32)

    xn = q8.double() * s8.double().repeat_interleave(128, 1)[:, :H]  # the norm itself has its own tests
    ref, slack = h.double().clone(), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for t in range(T):
        for k in range(K):
            e = int(idx[t, k])
            if e < 0:
                continue
            u = Wu[e] @ xn[t]
            s = u[I:] * torch.sigmoid(u[I:]) * u[:I]
            ref[t] += weight[t, k].double() * (Wd[e] @ s)
            slack[t] += weight[t, k].double() * (Wd[e].abs() @ s.abs())
    # the rows between the products are rounded to bf16, 2^-8 of each; the fp32 sums add far less
    assert ((out.double() - ref).abs() <= 2.0 ** -8 * 1.05 * slack + 1e-6 * ref.abs() + 1e-6).all()


@gpu
def test_layer_and_stack_over_int4_experts():
    """``Int4Experts`` under ``MoEStack`` against the layer in 64 bits with the same quantised weights."""
    from constellation_b200.context import MoEConfig, rms_norm
    from constellation_b200.int4 import Int4Experts, quantize_int4
    from constellation_b200.stack import MoEStack, StackLayer

    T, E, H, I = 20, 16, 256, 128
    cfg = MoEConfig(hidden_size=H, moe_intermediate_size=I, n_routed_experts=E, n_group=4, topk_group=2,
                    num_experts_per_tok=4)
    g = torch.Generator().manual_seed(7)
    layers, plain = [], []
    for _ in range(2):
        ex, W = Int4Experts("cuda", cfg, max_tokens=T), {}
        for e in [*range(E), -1]:
            parts = []
            for n, k in ((2 * I, H), (H, I)):
                w = (torch.randn(n, k, generator=g) * 0.05).cuda()
                q, s, z = quantize_int4(w)
                parts.append(((q, s, z), (torch.stack((q & 15, q >> 4), -1).view(n, k).double() - 8)
                              * s.double().repeat_interleave(128, 1)))
            ex.load_expert(e, parts[0][0], parts[1][0])
            W[e] = parts[0][1], parts[1][1]
        gate, bias = torch.randn(E, H, generator=g).cuda() * 0.1, torch.randn(E, generator=g).cuda() * 0.05
        layers.append(StackLayer(ex, gate, bias))
        plain.append(W)
    h0 = torch.randn(T, H, generator=g).to("cuda", torch.bfloat16)

    def expert(W, e, x):
        u = x @ W[e][0].T
        return (u[:, I:] * torch.sigmoid(u[:, I:]) * u[:, :I]) @ W[e][1].T

    h = h0
    for layer, W in zip(layers, plain):
        xn = rms_norm(h)
        out, idx, weight = layer.compute.moe_layer(xn, layer.gate_weight, layer.bias, residual=h, return_routes=True)
        ref = h.double() + expert(W, -1, xn.double())
        for k in range(4):
            for e in range(E):
                t = (idx[:, k] == e).nonzero().view(-1)
                ref[t] += weight[t, k, None].double() * expert(W, e, xn[t].double())
        # one rounding to bf16 of the result and one of the rows between the products
        assert ((out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -8 * ref.abs().amax(1, keepdim=True)).all()
        same = layer.compute.moe_routed_range(xn, idx, weight, 0, T, out_dtype=torch.float32)
        assert torch.equal(same, layer.compute.moe_routed(xn, idx, weight, add_shared=True, out_dtype=torch.float32))
        half = layer.compute.moe_routed_range(xn, idx, weight, 5, 9, out_dtype=torch.float32)
        bare = layer.compute.moe_routed(xn, idx, weight, out_dtype=torch.float32)
        assert torch.equal(half[5:9], same[5:9]) and torch.equal(half[:5], bare[:5]) and torch.equal(half[9:], bare[9:])
        h = out
    stack = MoEStack(layers, n_routed_experts=E)
    assert torch.equal(stack.forward(h0), h)
    for layer in layers:
        layer.compute.device_error()


@gpu
def test_two_halves_of_the_experts_add_up():
    from constellation_b200.context import MoEConfig
    from constellation_b200.int4 import Int4Experts, quantize_int4

    T, E, H, I = 12, 8, 128, 128
    cfg = MoEConfig(hidden_size=H, moe_intermediate_size=I, n_routed_experts=E, n_group=2, topk_group=2,
                    num_experts_per_tok=2)
    g = torch.Generator().manual_seed(3)
    whole = Int4Experts("cuda", cfg, max_tokens=T)
    parts = [Int4Experts("cuda", cfg, max_tokens=T, n_local=4, first_expert=b) for b in (0, 4)]
    for e in range(E):
        w = [quantize_int4((torch.randn(n, k, generator=g) * 0.05).cuda()) for n, k in ((2 * I, H), (H, I))]
        whole.load_expert(e, *w)
        parts[e // 4].load_expert(e, *w)
    x = torch.randn(T, H, generator=g).to("cuda", torch.float16)
    idx = torch.randint(0, E, (T, 2), generator=g).cuda()
    weight = torch.rand(T, 2, generator=g).cuda()
    one = whole.moe_routed(x, idx, weight, out_dtype=torch.float32)
    two = sum(p.moe_routed(x, idx, weight, out_dtype=torch.float32) for p in parts)
    assert ((one - two).abs() <= 4 * 2.0 ** -24 * (one.abs() + two.abs() + 1)).all()
    with pytest.raises(ValueError):
        parts[0].load_expert(5, *w)
    with pytest.raises(TypeError):
        whole.moe_routed(x.float(), idx, weight)


@gpu
def test_experts_from_the_reference_format():
    from constellation_b200.context import MoEConfig
    from constellation_b200.int4 import Int4Experts
    from oracle import cases
    from oracle.expert import DequantExpert

    H, I = 256, 128
    cfg = MoEConfig(hidden_size=H, moe_intermediate_size=I, n_routed_experts=2, n_group=1, topk_group=1,
                    num_experts_per_tok=1)
    ex = Int4Experts("cuda", cfg, max_tokens=4, group=32)
    b = cases.expert(5, H, I)
    ex.upload_expert(1, b.w_up, b.s_up, b.w_gate, b.s_gate, b.w_down, b.s_down)
    x = torch.from_numpy(cases.activations(6, 4, H)).to("cuda", torch.bfloat16)
    y = ex.moe_routed(x, torch.ones(4, 1, dtype=torch.int32, device="cuda"), torch.ones(4, 1, device="cuda"),
                      out_dtype=torch.float32)
    d = DequantExpert(b)
    up, gate = x.double() @ torch.from_numpy(d.w_up).cuda().double().T, x.double() @ torch.from_numpy(
        d.w_gate).cuda().double().T
    ref = (gate * torch.sigmoid(gate) * up) @ torch.from_numpy(d.w_down).cuda().double().T
    # 4-bit weights of groups of 32: a step is about 2.2 sigma / 7, its rounding 0.09 sigma a weight, in each of three
    # products in a row -- 0.16 of the result's size; 0.3 leaves room for chance, a wrong layout gives 1.4
    assert float((y.double() - ref).norm() / ref.norm()) < 0.3
    # expert 0 was not loaded: it gives zero
    assert (ex.moe_routed(x, torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.ones(4, 1, device="cuda")) == 0).all()


@gpu
def test_refusals_of_device_tensors():
    from constellation_b200 import _lib
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(2, 64, 256, 128, True)
    w, off = Int4Weight(q, s, z), offsets_of((2, 2))
    x, _, _ = make_x(4, 256, torch.bfloat16)
    x8, xs, _ = make_x(4, 256, torch.float8_e4m3fn)
    bad = [lambda: Int4Weight(q, s[:1], z), lambda: Int4Weight(q, s, z[:, :, :1]), lambda: Int4Weight(q, s[..., :0]),
           lambda: Int4Weight(q.int(), s, z), lambda: grouped_int4(x[:, :128], w, off), lambda: grouped_int4(x, w),
           lambda: grouped_int4(x, w, off.long()), lambda: grouped_int4(x, w, off[:2]),
           lambda: grouped_int4(x8, w, off), lambda: grouped_int4(x, w, off, x_scale=xs),
           lambda: grouped_int4(x8, w, off, x_scale=xs[:, :1]), lambda: grouped_int4(x, w, off.cpu()),
           lambda: grouped_int4(x, w, off, out=torch.empty(4, 63, device="cuda")),
           lambda: grouped_int4(x, w, off, out=torch.empty(4, 64, device="cuda"), out_dtype=torch.bfloat16),
           lambda: grouped_int4(x, w, off, out=x.view(-1)[:256].view(4, 64)),
           lambda: grouped_int4(x[:1].expand(2 ** 32 + 4, 256), w, off),
           lambda: grouped_int4(x.clone().requires_grad_(), w, off),
           lambda: grouped_int4(x8, w, off, x_scale=xs.clone().requires_grad_()),
           lambda: Int4Weight(q, s.clone().requires_grad_(), z)]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    for f in (lambda: grouped_int4(x.float(), w, off), lambda: grouped_int4(x[0], w, off),
              lambda: grouped_int4(x, w, off, out_dtype=torch.float64), lambda: Int4Weight(q.cpu(), s, z)):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(_lib.CstError):
        Int4Weight(q, torch.ones(2, 64, 256 // 16, device="cuda"))
    with pytest.raises(_lib.CstError):
        Int4Weight(q[:, :63], s[:, :63], z[:, :63], swiglu=True)
    with pytest.raises(IndexError):
        w.load(2, q[0], s[0], z[0])


def test_refusals_without_a_device():
    import ctypes

    from constellation_b200 import _lib
    from constellation_b200.int4 import Int4Weight, grouped_int4, quantize_int4

    with pytest.raises(TypeError):
        Int4Weight(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1))
    with pytest.raises(RuntimeError):
        Int4Weight.empty(1, 64, 128, device="cpu")
    with pytest.raises(TypeError):
        grouped_int4(torch.zeros(1, 128, dtype=torch.bfloat16), None)
    for bad in (16, 256):
        with pytest.raises(ValueError):
            quantize_int4(torch.zeros(4, 128), bad)
    q, s, z = quantize_int4(torch.linspace(-7, 7, 15).repeat(2, 9)[:, :128], 128)
    assert z is None and s.tolist() == [[1.0], [1.0]]
    assert ((torch.stack((q & 15, q >> 4), -1).view(2, 128).float() - 8) == torch.linspace(-7, 7, 15).repeat(2, 9)[:, :128]).all()
    L, P, BAD = _lib.lib, 16, _lib.CST_ERR_INVALID_ARG

    def weight(E=1, n=64, k=128, group=128, st=1, z=0, sw=0):
        return ctypes.byref(_lib.CstInt4Weight(E, n, k, group, st, z, sw))

    size = ctypes.c_int64()
    assert L.cst_int4_bytes(weight(), ctypes.byref(size)) == 0 and size.value == 8192 + 128 * 2 + 256
    assert L.cst_int4_bytes(weight(E=3, n=129, k=160, group=32, st=3, z=1), ctypes.byref(size)) == 0
    assert size.value == 3 * 2 * 2 * (8192 + 4 * 128 * 4 + 4 * 128) + 256
    for kw in (dict(E=0), dict(E=1025), dict(n=0), dict(k=0), dict(group=16), dict(k=130), dict(st=4), dict(n=3, sw=1),
               dict(n=1 << 21)):
        assert L.cst_int4_bytes(weight(**kw), ctypes.byref(size)) == BAD, kw
    assert L.cst_int4_bytes(None, ctypes.byref(size)) == BAD
    for a in ((None, P, None, P), (P, None, None, P), (P, P, None, None), (P, P, None, 8)):
        assert L.cst_int4_pack(weight(), 0, 1, *a, None) == BAD
    assert L.cst_int4_pack(weight(z=1), 0, 1, P, P, None, P, None) == BAD
    for first, count in ((-1, 1), (0, 3), (2, 1), (0, -1)):
        assert L.cst_int4_pack(weight(E=2), first, count, P, P, None, P, None) == BAD
    assert L.cst_int4_pack(weight(), 0, 0, None, None, None, None, None) == _lib.CST_OK
    assert L.cst_int4_device_error(weight(), None, None) == BAD

    assert L.cst_int4_workspace(weight(), 2, 3, ctypes.byref(size)) == 0 and size.value == 768 + 3 * 4
    assert L.cst_int4_workspace(weight(), 4, 3, ctypes.byref(size)) == 0 and size.value == 512 + 3 * 16
    for a in ((weight(), 3, 1), (weight(), 2, -1), (weight(group=16), 2, 1)):
        assert L.cst_int4_workspace(*a, ctypes.byref(size)) == BAD
    assert L.cst_int4_workspace(weight(), 2, 1, None) == BAD

    def call(w=None, data=P, x=P, xt=2, ldx=128, xs=None, lds=1, off=P, R=1, ws=P, out=P, ot=2, ldo=64):
        return L.cst_grouped_int4(w or weight(), data, x, xt, ldx, xs, lds, off, R, ws, out, ot, ldo, None)

    assert call(data=None, x=None, out=None, R=0) == _lib.CST_OK
    for kw in (dict(xt=3), dict(xt=4), dict(xs=P), dict(ot=4), dict(ldx=127), dict(ldo=63), dict(R=-1), dict(x=None),
               dict(out=None), dict(data=None), dict(w=weight(E=2), off=None), dict(xt=4, xs=P, lds=0),
               dict(ws=None), dict(ws=8), dict(data=8), dict(R=(1 << 28) + 1)):
        assert call(**kw) == BAD, kw
