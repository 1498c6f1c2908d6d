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
