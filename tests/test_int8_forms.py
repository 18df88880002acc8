"""Each kernel and tile of the products in 8-bit integers, asked for by kernel_configs: the form is seen to run, and its bits are those of the fp32
steps on the exact sum."""

import pytest
import torch

from tilegym_amd import _lib, ops

from .test_int8_ops import BF16, F16, F32, _check_matmul, _check_ragged, bits, codes, scales

RING = [(64, 32), (32, 64), (64, 64), (64, 128), (96, 128), (128, 128), (160, 128), (160, 192), (192, 192), (256, 128)]
TILE = dict(KERNEL="tiled")


def ran(**want):
    got = _lib.last_config()
    assert all(got[k] == v for k, v in want.items()), (got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("bm,bn", RING)
def test_ring_tiles(device, bm, bn):
    cfg = dict(KERNEL="tiled", BLOCK_M=bm, BLOCK_N=bn)
    # one tile and less, several with a rest in both directions; K of fewer steps than the ring has stages, of no whole step, and many
    for m, n, k in ((1, 8, 128), (bm, bn, 2048), (2 * bm + 5, 3 * bn - 24, 640), (bm - 1, bn + 8, 16), (bm + 17, 2 * bn, 1168), (3 * bm, bn + 40, 400)):
        for t, bias in ((BF16, None), (F32, None), (F16, F16)):
            _check_matmul(device, m, n, k, t, bias=bias, kernel_configs=cfg)
            ran(KERNEL=1, BLOCK_M=bm, BLOCK_N=bn, SPLIT_K=1)
    # outputs that are no whole vectors
    _check_matmul(device, bm + 3, bn + 5, 272, BF16, bias=F32, kernel_configs=cfg)
    _check_matmul(device, bm + 3, bn + 5, 272, F16, per_token=False, per_channel=False, kernel_configs=cfg)
    ran(KERNEL=1, BLOCK_M=bm, BLOCK_N=bn)


@pytest.mark.gpu
@pytest.mark.parametrize("bm,bn", RING)
@pytest.mark.parametrize("split", [2, 3, 8])
def test_ring_tiles_split(device, bm, bn, split):
    cfg = dict(KERNEL="tiled", BLOCK_M=bm, BLOCK_N=bn, SPLIT_K=split)
    for m, n, k in ((bm + 5, bn + 24, 2048), (17, 100, 1168), (33, 70, 1040)):
        _check_matmul(device, m, n, k, BF16, kernel_configs=cfg)
        _check_matmul(device, m, n, k, F32, bias=F32, per_token=False, kernel_configs=cfg)
        assert _lib.last_config()["SPLIT_K"] > 1


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(256, 256, 256), (1, 8, 256), (257, 264, 384), (700, 1000, 1024), (512, 512, 4096), (3000, 5128, 256)])
def test_tile256(device, m, n, k):
    cfg = dict(KERNEL="tiled", BLOCK_M=256, BLOCK_N=256)
    for t, bias in ((BF16, None), (F32, F32), (F16, None)):
        _check_matmul(device, m, n, k, t, bias=bias, kernel_configs=cfg)
        ran(KERNEL=1, BLOCK_M=256, BLOCK_N=256)
    _check_matmul(device, m, n, k, BF16, bias=BF16, per_token=False, per_channel=False, kernel_configs=cfg)
    _check_matmul(device, m, n, k, F16, bias=F16, kernel_configs=cfg)


@pytest.mark.gpu
def test_tile256_more_tiles_than_compute_units(device):
    """Workgroups that walk several tiles, with rows and columns left over."""
    _check_matmul(device, 4097, 8200, 384, BF16, kernel_configs=dict(KERNEL="tiled", BLOCK_M=256, BLOCK_N=256))
    ran(KERNEL=1, BLOCK_M=256, BLOCK_N=256)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 20, 24, 40, 56, 64])
def test_stream(device, rows):
    cfg = dict(KERNEL="stream", BLOCK_N=rows)
    for m, n, k in ((1, 8, 16), (16, 300, 512), (5, 1000, 1024), (17, 264, 4096), (32, 72, 1552), (31, 333, 2064), (7, 64, 400)):
        for t, bias in ((BF16, None), (F32, F32), (F16, None)):
            _check_matmul(device, m, n, k, t, bias=bias, kernel_configs=cfg)
            ran(KERNEL=3, BLOCK_N=rows, SPLIT_K=1)
        if k > 1024:
            _check_matmul(device, m, n, k, BF16, per_token=False, kernel_configs=dict(cfg, SPLIT_K=3))
            assert _lib.last_config()["SPLIT_K"] > 1


@pytest.mark.gpu
def test_simple(device):
    cfg = dict(KERNEL="fallback")
    for m, n, k in ((1, 1, 1), (64, 64, 64), (100, 200, 300), (65, 8, 4096)):
        _check_matmul(device, m, n, k, BF16, kernel_configs=cfg)
        ran(KERNEL=0)


COUNTS = [[5, 0, 70, 1], [16, 17, 0, 33, 260], [0, 0, 300], [1] * 70, [0] * 150 + [40] + [3] * 20]


@pytest.mark.gpu
@pytest.mark.parametrize("bm,bn", RING)
def test_ragged_ring_tiles(device, bm, bn):
    cfg = dict(KERNEL="tiled", BLOCK_M=bm, BLOCK_N=bn)
    for counts in COUNTS:
        for n, k in ((bn + 24, 640), (40, 144)):
            _check_ragged(device, counts, n, k, BF16, tail=9, start=3, kernel_configs=cfg)
            ran(KERNEL=1, BLOCK_M=bm, BLOCK_N=bn)
    _check_ragged(device, [5, 2 * bm + 1, 0, 3], bn + 5, 272, F32, tail=1, kernel_configs=cfg)


@pytest.mark.gpu
def test_ragged_tile256(device):
    cfg = dict(KERNEL="tiled", BLOCK_M=256, BLOCK_N=256)
    for counts in COUNTS + [[0] * 70, [300, 0, 257, 256, 255, 1] * 50]:  # (the last: several tiles for a workgroup, experts beyond its first 64 and 256)
        for n, k in ((280, 640), (40, 256)):
            for t in (BF16, F32, F16):
                _check_ragged(device, counts, n, k, t, tail=9, start=3, kernel_configs=cfg)
                ran(KERNEL=1, BLOCK_M=256, BLOCK_N=256)
    _check_ragged(device, [0] * 63 + [600, 900] + [0] * 63 + [700] + [0] * 100 + [1], 3000, 384, BF16, tail=300, start=0, kernel_configs=cfg)
    _check_ragged(device, [5, 513, 0, 3], 264, 272, F32, tail=1, kernel_configs=cfg)  # K in no whole steps: another form
    assert _lib.last_config()["BLOCK_N"] != 256


@pytest.mark.gpu
def test_ragged_stream_and_simple(device):
    for counts in COUNTS:
        for n, k in ((200, 1024), (40, 400), (72, 16)):
            for t in (BF16, F32):
                _check_ragged(device, counts, n, k, t, tail=9, start=3, kernel_configs=dict(KERNEL="stream", BLOCK_N=64))
                ran(KERNEL=3)
                _check_ragged(device, counts, n, k, t, tail=9, start=3, kernel_configs=dict(KERNEL="fallback"))
                ran(KERNEL=0)


@pytest.mark.gpu
def test_forms_that_do_not_take_a_problem_are_ignored(device):
    _check_matmul(device, 40, 64, 100, BF16, kernel_configs=dict(KERNEL="tiled", BLOCK_M=128, BLOCK_N=128))  # rows of 100 bytes
    ran(KERNEL=0)
    _check_matmul(device, 40, 68, 256, BF16, kernel_configs=dict(KERNEL="tiled", BLOCK_M=256, BLOCK_N=256))  # outputs in no whole vectors
    _check_matmul(device, 40, 64, 256, BF16, kernel_configs=dict(KERNEL="stream"))                           # more rows than it takes
    _check_matmul(device, 40, 64, 256, BF16, kernel_configs=dict(KERNEL="tiled", BLOCK_M=48, BLOCK_N=128))


@pytest.mark.gpu
def test_ragged_offsets_beyond_the_rows(device):
    """Whatever indptr holds, every form stays within the rows."""
    a, b = codes((50, 128), 1).to(device), codes((3, 64, 128), 2).to(device)
    sa, sb = scales(50, 3).to(device), scales((3, 64), 4).to(device)
    want = ops.ragged_int8_matmul(a, b, sa, sb, torch.tensor([0, 20, 40, 50], dtype=torch.int32, device=device))
    for cfg in [dict(KERNEL="tiled", BLOCK_M=m, BLOCK_N=n) for m, n in RING] + [dict(KERNEL="stream"), dict(KERNEL="fallback")]:
        got = torch.zeros(50, 64, dtype=BF16, device=device)
        ops.ragged_int8_matmul(a, b, sa, sb, torch.tensor([0, 20, 40, 500], dtype=torch.int32, device=device), out=got, kernel_configs=cfg)
        assert torch.equal(bits(got[:40]), bits(want[:40]))
        ops.ragged_int8_matmul(a, b, sa, sb, torch.tensor([-5, 20, 10, 40], dtype=torch.int32, device=device), out=got, kernel_configs=cfg)
