"""The form that an int8 product takes: the same with the scratch memory that it asked for as with any amount, and every part of a split K with a share of it."""

import ctypes
import random

import pytest
import torch

from tilegym_amd import _lib, ops

from .test_int8_ops import BF16, bits, codes, scales


def form_of(m, n, k, room, kernel_configs=None):
    """(kernel, BLOCK_M, BLOCK_N, parts of K)."""
    out, (cfg, ncfg) = (ctypes.c_int32 * 4)(), _lib.make_cfg(kernel_configs)
    assert _lib.load().tg_diag_int8_gemm_form(m, n, k, room, cfg, ncfg, out) == 0
    return tuple(out)


def needed(m, n, k, kernel_configs=None):
    return _lib.load().tg_int8_gemm_workspace_bytes(m, n, k, *_lib.make_cfg(kernel_configs))


def test_form_query_needs_no_device():
    query, (cfg, ncfg), out = _lib.load().tg_diag_int8_gemm_form, _lib.make_cfg(None), (ctypes.c_int32 * 4)()
    for m, n, k in ((0, 8, 64), (4, 0, 64), (4, 8, 0), (4, 8, 131072), (2 ** 31, 8, 64)):
        assert query(m, n, k, 0, cfg, ncfg, out) == -6
    assert query(4, 8, 64, 0, cfg, ncfg, None) == -5
    assert form_of(4096, 4096, 4096, 0)[0] == 1 and form_of(1, 4096, 4096, 0)[0] == 3 and form_of(1, 4096, 4097, 0)[0] == 0


FORCED = [dict(KERNEL="fallback"), dict(KERNEL="tiled", BLOCK_M=64, BLOCK_N=64, SPLIT_K=8), dict(KERNEL="tiled", BLOCK_M=32, BLOCK_N=64, SPLIT_K=5),
          dict(KERNEL="stream", SPLIT_K=8), dict(KERNEL="stream", BLOCK_N=32, SPLIT_K=3)]


@pytest.mark.parametrize("aligned", [True, False])
def test_what_is_planned_runs(aligned):
    """With exactly the bytes that a problem asks for the form is the one that unlimited scratch memory leads to."""
    rng, split, uneven = random.Random(int(aligned)), 0, 0
    cases = [(1, 512, 4480), (1, 512, 4224), (16, 1024, 13824), (64, 1024, 5376)] if aligned else [(1, 513, 4201), (200, 600, 16001), (1, 4478, 13250)]
    while len(cases) < 4000:
        m, n, k = round(2 ** rng.uniform(0, 10)), round(2 ** rng.uniform(3, 14)), round(2 ** rng.uniform(8, 15))
        cases.append((m, n // 8 * 8, k // 128 * 128 + 128 * (rng.random() < 0.5) + 16 * rng.randint(0, 7)) if aligned else (m, n, k | 1))
    for i, (m, n, k) in enumerate(cases):
        for cfg in (None, FORCED[i % len(FORCED)]):
            plan, bytes_ = form_of(m, n, k, 2 ** 62, cfg), needed(m, n, k, cfg)
            kernel, _, _, parts = plan
            assert bytes_ == (parts * m * n * 4 if parts > 1 else 0), (m, n, k, cfg)
            assert form_of(m, n, k, bytes_, cfg) == plan, (m, n, k, cfg)
            assert form_of(m, n, k, bytes_ + 12345, cfg) == plan, (m, n, k, cfg)
            units = -(-k // (512 if kernel == 3 else 128))
            assert (parts - 1) * -(-units // parts) < units, (m, n, k, cfg)   # the last part has a step
            if cfg is None:
                split, uneven = split + (parts > 1), uneven + (parts > 1 and parts not in (2, 4, 8))
    assert split > 200 and (uneven == 0 if aligned else uneven > 50)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 512, 4480), (1, 512, 4224), (16, 1024, 13824), (64, 1024, 5376), (1, 513, 4201), (5, 4478, 13250)])
def test_calls_run_what_was_planned(device, m, n, k):
    a, b, sa, sb = codes((m, k), 1).to(device), codes((n, k), 2).to(device), scales(m, 3).to(device), scales(n, 4).to(device)
    got = ops.int8_matmul(a, b, sa, sb)
    ran = _lib.last_config()
    assert (ran["KERNEL"], ran["BLOCK_M"], ran["BLOCK_N"], ran["SPLIT_K"]) == form_of(m, n, k, 2 ** 62)
    want = ((a.double() @ b.double().t()).float() * sa[:, None] * sb).to(BF16)
    assert torch.equal(bits(got), bits(want))
