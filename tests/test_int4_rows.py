"""The rows of 4-bit products: their scales, their workspace and what lies around them.

Bounds are those of ``test_int4.check``: the sums' rounding, and one rounding of the result.
"""
import pytest
import torch

from test_int4 import check, make_weight, make_x, offsets_of

gpu = pytest.mark.gpu


def product_in(room, x, w, offsets, out_dtype=torch.float32):
    """``grouped_int4`` through the C entry, in a workspace whose former contents are the caller's."""
    from constellation_b200 import _lib
    from constellation_b200.context import dtype_code

    R = x.shape[0]
    out = torch.empty(R, w.out_features, dtype=out_dtype, device="cuda")
    assert room.numel() >= w._workspace(dtype_code(x.dtype), R)
    _lib.check(_lib.lib.cst_grouped_int4(
        w._ref, w.data.data_ptr(), x.data_ptr(), dtype_code(x.dtype), x.stride(0), None, 0,
        None if offsets is None else offsets.data_ptr(), R, room.data_ptr(), out.data_ptr(), dtype_code(out_dtype),
        w.out_features, torch.cuda.current_stream().cuda_stream))
    return out


def rows_of_every_size(R, K, dt, seed=1):
    """Rows whose largest lie in different binades, each starting off a 16-byte boundary (such rows are read
    element by element, so that the split takes long)."""
    x, _, _ = make_x(R, K, torch.float32, seed)
    power = torch.arange(R) * 5 % 17 - 8 if dt == torch.float16 else torch.arange(R) * 7 % 41 - 20
    wide = torch.empty(R, K + 3, dtype=dt, device="cuda")
    wide[:, 1:K + 1] = x * torch.exp2(power.float().clamp(max=12).cuda())[:, None]
    return wide[:, 1:K + 1]


# one weight and a few rows: k is split over a cluster, whose last CTAs have no steps of it
SPLITS = [(8, 2048, 2560, 128, False, torch.bfloat16), (8, 1024, 5120, 128, False, torch.bfloat16),
          (8, 1536, 3584, 128, False, torch.bfloat16), (8, 4096, 2304, 128, False, torch.bfloat16),
          (16, 2048, 7168, 128, False, torch.bfloat16), (32, 512, 7168, 128, False, torch.bfloat16),
          (20, 136, 1152, 128, False, torch.bfloat16), (32, 256, 1152, 64, True, torch.float16),
          (8, 2816, 2048, 128, False, torch.float16)]


@gpu
@pytest.mark.parametrize("R,N,K,group,zeros,dt", SPLITS)
def test_row_scales_of_a_split_k(R, N, K, group, zeros, dt):
    """Every row's own scale, whatever the workspace held: a CTA without products has to wait for them too."""
    from constellation_b200.int4 import Int4Weight

    q, s, z, W = make_weight(1, N, K, group, zeros)
    w = Int4Weight(q, s, z)
    x = rows_of_every_size(R, K, dt)
    room = torch.empty(w._workspace(1 if dt == torch.float16 else 2, R), dtype=torch.uint8, device="cuda")
    for byte in (0xFF, 0x47, 0xFF):  # NaN, then scales of 5e4, in the scales' place
        room.fill_(byte)
        check(product_in(room, x, w, None), x.double(), W, None, group, False)


@gpu
def test_ctas_without_products_between_products():
    """A grid is sized for rows of every expert: with all rows at one expert most CTAs find no item, with none at any all
    do, and they give their tensor memory back to the products that follow."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    E, N, K, R = 64, 256, 384, 48
    weights = [make_weight(E, N, K, 128, zeros) for zeros in (False, True)]
    held = [Int4Weight(q, s, z) for q, s, z, _ in weights]
    x, _, x64 = make_x(R, K, torch.bfloat16)
    ragged = [R * e // E for e in range(E + 1)]
    orders = [torch.tensor(off, dtype=torch.int32, device="cuda")
              for off in ([0] * 7 + [R] * (E - 6), [0] * (E + 1), ragged)]
    got = [(i, off, grouped_int4(x, held[i], off, out_dtype=torch.float32))
           for _ in range(8) for off in orders for i in range(2)]
    for i, off, out in got:
        check(out, x64, weights[i][3], off, 128, False)
    for w in held:
        w.device_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses stay on machines that could not launch a kernel")
def test_an_out_that_overlaps_an_input_is_refused():
    """By address alone, so nothing is read, written or launched; what is refused lies at made-up addresses."""
    import ctypes

    from constellation_b200 import _lib

    L, BAD, MB = _lib.lib, _lib.CST_ERR_INVALID_ARG, 1 << 20
    w = ctypes.byref(_lib.CstInt4Weight(2, 64, 256, 128, 1, 0, 0))
    size = ctypes.c_int64()
    assert L.cst_int4_bytes(w, ctypes.byref(size)) == 0
    data = size.value
    assert L.cst_int4_workspace(w, 4, 8, ctypes.byref(size)) == 0
    room = size.value

    def call(out, ldo=64, ot=2, xt=4, ldx=256, lds=2):
        xs = 2 * MB if xt == 4 else None
        rc = L.cst_grouped_int4(w, 4 * MB, MB, xt, ldx, xs, lds, 3 * MB, 8, 5 * MB, out, ot, ldo, None)
        return rc == BAD and b"overlaps" in L.cst_last_error()

    # out takes 8 * 64 * 2 bytes
    for first, last in ((MB, MB + 8 * 256), (2 * MB, 2 * MB + 8 * 2 * 4), (3 * MB, 3 * MB + 3 * 4),
                        (4 * MB, 4 * MB + data), (5 * MB, 5 * MB + room)):
        for out in (first - 1024 + 2, first, last - 2):
            assert call(out)
    assert call(MB + 300, ldx=512)  # from the gap behind a row on, at another pitch
    # columns of one array of 1024 bytes a row: x (bf16, 512 bytes) at 0 (and one where rows wrap into it)
    for out in (MB + 510, MB - 1024 + 900, MB + 1024 * 7 + 510):
        assert call(out, ldo=512, xt=2, ldx=512)


@gpu
def test_out_beside_the_inputs():
    """Next to its inputs in one buffer an out is taken, on top of any of them it is not."""
    from constellation_b200 import _lib
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(2, 64, 256, 128, False)
    w, off = Int4Weight(q, s), offsets_of((3, 4))
    x, xs, x64 = make_x(8, 256, torch.float8_e4m3fn)
    want = grouped_int4(x, w, off, x_scale=xs)
    buf = torch.zeros(16384, dtype=torch.uint8, device="cuda")

    def put(at, t):
        buf[at:at + t.numel() * t.element_size()] = t.contiguous().view(torch.uint8).view(-1)
        return buf[at:at + t.numel() * t.element_size()].view(t.dtype).view(t.shape)

    # x 2048 bytes, its scales 64, offsets 12, out 1024
    x1, xs1, off1 = put(1024, x), put(3200, xs), put(3264, off)
    for at in (0, 3280):
        out = buf[at:at + 1024].view(torch.bfloat16).view(8, 64)
        assert torch.equal(grouped_int4(x1, w, off1, x_scale=xs1, out=out), want)
    for at in (16, 1024, 2048, 3184, 3248, 3264):
        out = buf[at:at + 1024].view(torch.bfloat16).view(8, 64)
        with pytest.raises(RuntimeError, match="overlaps"):
            grouped_int4(x1, w, off1, x_scale=xs1, out=out)
    # other columns of x's array
    xb, _, xb64 = make_x(8, 256, torch.bfloat16)
    wide = torch.zeros(8, 320, dtype=torch.bfloat16, device="cuda")
    wide[:, :256] = xb
    room = torch.empty(w._workspace(2, 8), dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib.cst_grouped_int4(w._ref, w.data.data_ptr(), wide.data_ptr(), 2, 320, None, 0, off.data_ptr(), 8,
                                         room.data_ptr(), wide.data_ptr() + 512, 2, 320,
                                         torch.cuda.current_stream().cuda_stream))
    assert torch.equal(wide[:, 256:], grouped_int4(xb, w, off)) and torch.equal(wide[:, :256], xb)


def check_chunks(out, x, W, group, dt):
    """Against W x in 64 bits: the sums' rounding, and what terms may drop of a number, which goes by the largest of its
    128 columns.  Terms fit the largest of a row to 448 and drop at most 2^-14 of their power of two (bf16: half of
    e4m3's smallest step of 2^-9, over 16; fp16: the third term is 512 times a rest below 2^-10, and rounded to half a
    step of 2^-5: 2^-15).  A chunk takes its own where its largest is 5 binades below, so its power of two is at most
    2^4 times the smallest that fits its largest, which is above 224 of that: 2^-14 * 2^4 / 224 < 2^-17."""
    K, x64 = W.shape[1], x.double()
    most = torch.stack([c.abs().amax(1) for c in x64.split(128, 1)], 1)
    sizes = torch.stack([c.abs().sum(1) for c in W.split(128, 1)], 1)
    ref = x64 @ W.T
    err = (group + 2 * K / group + 64) * 2.0 ** -23 * (x64.abs() @ W.abs().T) + 2.0 ** -17 * (most @ sizes.T)
    bound = err + ref.abs() * 2.0 ** -24 + 2.0 ** -126
    got = out.double()
    assert ((got - ref).abs() <= bound).all(), ((got - ref).abs() / bound).max()


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,N,K,group,zeros", [(1, 136, 640, 128, False), (8, 2048, 2560, 128, False),
                                               (13, 200, 1152, 64, True), (40, 144, 2048, 128, True),
                                               (70, 96, 864, 32, False), (5, 64, 10240, 128, False),
                                               (600, 1024, 1024, 128, False)])
def test_an_outlier_costs_the_others_nothing(R, N, K, group, zeros, dt):
    """Numbers 10^4.8 times the rest in a group of weights that is all zero: what is left are the other columns, and they
    have as many bits as if the outlier were not there."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(1, N, K, group, zeros)
    at = K // 2 // 128 * 128  # a chunk's first column, and the groups of that chunk
    s[:, :, at // group:(at + 128) // group] = 0
    W[:, :, at:at + 128] = 0
    w = Int4Weight(q, s, z)
    x, _, _ = make_x(R, K, torch.float32)
    plain = x.to(dt)
    x[:, at + 3] = 60000.0
    x[::3, at + 40] = -3000.0
    if R > 2:
        x[1, at + 3] = 0.5  # a row without one
        x[2] *= 2.0 ** -6
        x[2, 128:] *= 2.0 ** -7  # and one whose chunks differ
        plain[1:3] = x[1:3].to(dt)
    x = x.to(dt)
    out = grouped_int4(x, w, out_dtype=torch.float32)
    check_chunks(out, x, W[0], group, dt)
    assert torch.equal(grouped_int4(x, w, out_dtype=torch.float32), out)
    if R > 2:  # rows do not depend on the rows beside them
        plain[0] = plain[1]
        plain[2] = plain[1]
        assert torch.equal(grouped_int4(plain, w, out_dtype=torch.float32)[1], out[1])


@gpu
@pytest.mark.parametrize("factor", [2.0 ** 30, 2.0 ** 90, 2.0 ** 120])
def test_chunks_of_every_size_in_a_row(factor):
    """bf16 chunks far apart, beside chunks of zeros: each keeps its bits where the larger ones' weights are zero."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    N, K, R = 96, 1024, 11
    q, s, z, W = make_weight(1, N, K, 128, False, torch.float32)
    x, _, _ = make_x(R, K, torch.float32)
    x[:, 256:384] *= factor
    x[:, 512:640] /= factor
    x[::2, 768:896] = 0
    x = x.to(torch.bfloat16)
    for held in ([0, 1, 3, 4, 5, 6, 7], [4], [2], [2, 4, 6]):
        keep = torch.zeros(K // 128, dtype=torch.bool)
        keep[held] = True
        s1 = torch.where(keep.cuda(), s, torch.zeros((), device="cuda"))
        W1 = W * keep.cuda().double().repeat_interleave(128)
        out = grouped_int4(x, Int4Weight(q, s1, z), out_dtype=torch.float32)
        assert torch.isfinite(out).all()
        check_chunks(out, x, W1[0], 128, torch.bfloat16)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_outliers_among_experts(dt):
    """Experts of one and of many rows with and without outliers, NaN in a row, and rows of no expert full of both."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    counts, N, K = (3, 0, 40, 9, 1, 17), 160, 1280
    q, s, z, W = make_weight(len(counts), N, K, 128, True)
    w, off, R = Int4Weight(q, s, z), offsets_of(counts), sum(counts)
    x, _, _ = make_x(R + 4, K, torch.float32)
    x[::5, 700] = 9000.0
    x[R:] = 1e-6
    x[R:, 5] = 60000.0
    x = x.to(dt)
    clean = grouped_int4(x, w, off, out_dtype=torch.float32)
    assert (clean[R:] == 0).all()
    for e, (lo, hi) in enumerate(zip(off.tolist(), off.tolist()[1:])):
        if hi > lo:
            # zero points take part in the sums, so that their magnitude is that of scale (q + zero) |x|
            most = x[lo:hi].double().abs()
            v = torch.stack((q[e] & 15, q[e] >> 4), -1).view(N, K).double() + z[e].double().repeat_interleave(128, 1)
            mag = v * s[e].double().repeat_interleave(128, 1)
            ref = x[lo:hi].double() @ W[e].T
            bound = (128 + 2 * K / 128 + 64) * 2.0 ** -23 * (most @ mag.T) + 2.0 ** -17 * (
                torch.stack([c.amax(1) for c in most.split(128, 1)], 1)
                @ torch.stack([c.abs().sum(1) for c in W[e].split(128, 1)], 1).T) + ref.abs() * 2.0 ** -24
            assert ((clean[lo:hi].double() - ref).abs() <= bound).all()
    x[7, 3], x[48, 1279] = float("nan"), float("inf")
    out = grouped_int4(x, w, off, out_dtype=torch.float32)
    keep = [r for r in range(R) if r not in (7, 48)]
    assert torch.equal(out[keep], clean[keep]) and not torch.isfinite(out[[7, 48]]).any()


@gpu
@pytest.mark.parametrize("outlier", [False, True])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_items_one_after_the_other_in_a_cluster(dt, outlier):
    """160 items of 21 steps over pairs of CTAs: a pair's sums of one item lie beside those of the next."""
    from constellation_b200.int4 import Int4Weight

    R, N, K = 40, 10240, 5376
    q, s, z, W = make_weight(1, N, K, 128, False)
    s[:, :, 20] = 0
    W[:, :, 2560:2688] = 0
    w = Int4Weight(q, s, z)
    x = rows_of_every_size(R, K, dt)
    if outlier:
        x[:, 2600] = x.abs().amax(1) * (40.0 if dt == torch.float16 else 2.0 ** 17)
    room = torch.full((w._workspace(1 if dt == torch.float16 else 2, R),), 0xFF, dtype=torch.uint8, device="cuda")
    out = product_in(room, x, w, None)
    check_chunks(out, x, W[0], 128, dt)
    for _ in range(3):
        assert torch.equal(product_in(room, x, w, None), out)


@gpu
def test_outliers_that_come_and_go_between_replays():
    """Captured calls in two graphs on two streams at once, whose rows change between replays, and eager calls beside."""
    from constellation_b200.int4 import Int4Weight, grouped_int4

    q, s, z, W = make_weight(4, 512, 2048, 128, True)
    w, off = Int4Weight(q, s, z), offsets_of((5, 0, 20, 2))
    plain, _, _ = make_x(30, 2048, torch.bfloat16)
    spiky = plain.clone()
    spiky[::4, 77] = 2.0 ** 16
    want = [grouped_int4(x, w, off, out_dtype=torch.float32) for x in (plain, spiky)]
    xs, graphs, outs = [plain.clone(), spiky.clone()], [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(grouped_int4(x, w, off, out_dtype=torch.float32))
    streams = [torch.cuda.Stream() for _ in xs]
    for turn in range(6):
        for i, x in enumerate(xs):
            x.copy_((plain, spiky)[(i + turn) % 2])
        torch.cuda.synchronize()
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                graphs[i].replay()
        beside = grouped_int4(spiky, w, off, out_dtype=torch.float32)
        torch.cuda.synchronize()
        assert torch.equal(beside, want[1])
        assert all(torch.equal(outs[i], want[(i + turn) % 2]) for i in range(2)), turn
    w.device_error()
