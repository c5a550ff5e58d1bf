"""Layer norm between column blocks of one wider buffer: apart where the rows have one stride and no column is in both, refused (in front of any launch) otherwise."""
import pytest
import torch

from encodermap_amd import _lib

P = 1 << 20    # an address that nothing reads
CLOSE = [       # (y - x in elements, stride of x, of y) of eight columns that meet
    (7, 20, 20), (13, 20, 20), (19, 20, 20), (1, 20, 20), (20, 20, 20), (-7, 20, 20), (-13, 20, 20), (-20, 20, 20), (8, 15, 15), (8, 20, 21), (8, 20, 40), (7, 0, 20),
    (20 * 2 + 7, 20, 20), (-20 * 2 + 5, 20, 20)]


@pytest.mark.parametrize("ahead,ldx,ldy", CLOSE)
def test_columns_of_both_are_refused(ahead, ldx, ldy):
    lib = _lib.load()
    x, y = P, P + 4 * ahead
    assert lib.emx_layernorm_fwd(x, 0, 4, 8, ldx, None, None, 1e-3, y, ldy, None, None, None) == -1
    assert b"overlap" in lib.emx_last_error()
    ws = _lib.layernorm_ws_floats(4, 8)
    for dy, xx, ld_dy, ld_x in ((x, 9 * P, ldx, 8), (9 * P, x, 8, ldx)):
        assert lib.emx_layernorm_bwd(dy, ld_dy, xx, ld_x, 0, 4, 8, None, 3 * P, 4 * P, y, ldy, None, None, 5 * P, ws, None) == -1
        assert b"overlap" in lib.emx_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D,gap", [(8, 0), (70, 3), (128, 0), (1000, 5), (20000, 1)])
def test_column_blocks_of_one_buffer(D, gap, kind):
    _lib.require_gpu()
    dtype, n = getattr(torch, kind), 45
    gen = torch.Generator("cuda").manual_seed(D)
    wide = torch.randn(n + 1, 4 * D + 3 * gap + 2, generator=gen, device="cuda").to(dtype)
    gamma, beta = torch.randn(D, generator=gen, device="cuda"), torch.randn(D, generator=gen, device="cuda")
    blocks = [wide[:n, i * (D + gap):i * (D + gap) + D] for i in range(3)] + [wide[1:, 3 * (D + gap):3 * (D + gap) + D]]     # (the last one a row further down)
    outside = wide.clone()
    x, dy = blocks[1].clone(), blocks[2].clone()
    y, dx = torch.empty_like(x), torch.empty_like(x)
    stats, grads = [torch.empty(n, device="cuda") for _ in range(2)], [torch.empty(D, device="cuda") for _ in range(2)]
    ws = torch.empty(_lib.layernorm_ws_floats(n, D), device="cuda")
    _lib.layernorm_fwd(x, gamma, beta, 1e-3, y, *stats)
    _lib.layernorm_bwd(dy, x, gamma, *stats, dx, *grads, ws)
    got_stats, got_grads = [torch.empty(n, device="cuda") for _ in range(2)], [torch.empty(D, device="cuda") for _ in range(2)]
    _lib.layernorm_fwd(blocks[1], gamma, beta, 1e-3, blocks[0], *got_stats)
    _lib.layernorm_bwd(blocks[2], blocks[1], gamma, *got_stats, blocks[3], *got_grads, ws)
    assert torch.equal(blocks[0], y) and torch.equal(blocks[3], dx)
    assert all(torch.equal(a, b) for a, b in zip(stats + grads, got_stats + got_grads))
    for b in (outside, wide):
        b[:n, :D] = 0
        b[1:, 3 * (D + gap):3 * (D + gap) + D] = 0
    assert torch.equal(wide, outside)
