"""A NaN in a product stays a NaN through every activation: the microscaled products, gated ones, and gz_gemm_run_ex.

relu(NaN) is NaN by its formula as used throughout (x where x > 0 or x is NaN, else 0), so what a block's NaN
scale, a NaN or an infinity among the values says about a result is not lost behind it."""
import numpy as np
import pytest
import torch

import gemm_zoo_b200 as gz
from gemm_zoo_b200 import api
from tests import mx_oracle as orc
from tests.test_microscale import ACTS, FP4, NV, _mx

pytestmark = pytest.mark.gpu


def _poison(q, row):
    """A NaN scale in the first block of a row."""
    groups = -(-(-(-q.k // orc.block(q.format))) // 4)
    q.scales[(row // 128 * groups) * 512 + (row % 32) * 16 + (row % 128 // 32) * 4] = 255 if q.format == FP4 else 127


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("fmt", [FP4, NV])
@pytest.mark.parametrize("config,m", [(gz.MX_CFG_SWAP_M16, 1), (gz.MX_CFG_SWAP_M64, 40), (gz.MX_CFG_SINGLE, 130),
                                      (gz.MX_CFG_SINGLE_N128, 130), (gz.MX_CFG_PAIR, 300), (gz.MX_CFG_PAIR_N128, 300)])
def test_nan_of_a_row_and_of_a_column(act, fmt, config, m):
    n, k, r, c = 200, 300, m - 1, 77
    (a, av), (b, bv) = _mx(m, k, fmt, 1, True), _mx(n, k, fmt, 2, True)
    _poison(a, r), _poison(b, c)
    for dtype in (torch.float32, torch.bfloat16):
        d = torch.zeros(m, n, dtype=dtype, device="cuda")
        gz.MxGemm(m, n, k, fmt, dtype, config=config)(a, b, None, d, 1.0, 0.0, activation=ACTS[act])
        want = np.zeros((m, n), dtype=bool)
        want[r], want[:, c] = True, True
        assert np.array_equal(torch.isnan(d).cpu().numpy(), want)
        if act == "relu" and dtype == torch.float32:
            assert np.array_equal(d.cpu().double().numpy()[~want], np.maximum(av @ bv.T, 0)[~want])


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("out", [torch.float32, torch.float16, FP4, NV])
@pytest.mark.parametrize("config,m", [(gz.MX_CFG_SWAP_M16, 9), (gz.MX_CFG_SINGLE, 130), (gz.MX_CFG_PAIR, 200)])
def test_nan_of_the_gate_alone_and_of_up_alone(act, out, config, m):
    n, k, cg, cu = 200, 64, 77, 150
    a, _ = _mx(m, k, NV, 1, True)
    (g, _), (u, _) = _mx(n, k, NV, 2, True), _mx(n, k, NV, 3, True)
    _poison(g, cg), _poison(u, cu)
    plan = gz.MxGated(m, n, k, NV, out, activation=ACTS[act], config=config)
    if isinstance(out, torch.dtype):
        d = torch.zeros(m, n, dtype=out, device="cuda")
        plan(a, g, u, d, 2.0 ** -4, 2.0 ** -4)
        got = torch.isnan(d).cpu().numpy()
        size = 1
    else:
        q = gz.MxMatrix.empty(m, n, out)
        plan(a, g, u, q, 2.0 ** -4, 2.0 ** -4)
        got = torch.isnan(gz.mx_dequantize(q, torch.empty(m, n, device="cuda"))).cpu().numpy()
        size = orc.block(out)
    want = np.zeros((m, n), dtype=bool)
    for c in (cg, cu):
        want[:, c // size * size:(c // size + 1) * size] = True
    assert np.array_equal(got, want)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_nan_and_infinity_among_the_values(value):
    x, w = torch.randn(40, 256, device="cuda"), torch.randn(96, 256, device="cuda")
    x[3, 100] = value
    d = torch.empty(40, 96, device="cuda")
    for fmt in (FP4, NV):
        gz.MxGemm(40, 96, 256, fmt, torch.float32)(gz.mx_quantize(x, fmt), gz.mx_quantize(w, fmt), None, d, 1.0, 0.0,
                                                   activation=gz.ACT_RELU)
        bad = torch.isnan(d).cpu()
        assert bool(bad[3].all()) and not bool(bad[:3].any()) and not bool(bad[4:].any())


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("config,m", [(gz.CFG_AUTO, 300), (gz.CFG_1CTA_N128, 300), (gz.CFG_2CTA_N256, 300),
                                      (gz.CFG_2CTA_M512_N256, 700), (gz.CFG_SWAP_M64, 64), (gz.CFG_SIMT, 70)])
def test_nan_through_the_epilogue_of_the_16_bit_products(act, config, m):
    n, k, r, c = 200, 128, m - 1, 77
    rng = np.random.default_rng(m)
    a = torch.from_numpy(rng.integers(-3, 4, (m, k)).astype(np.float32)).to(torch.bfloat16).cuda()
    b = torch.from_numpy(rng.integers(-3, 4, (n, k)).astype(np.float32)).to(torch.bfloat16).cuda()
    a[r, 5], b[c, 9] = float("nan"), float("nan")
    g = gz.Sm100Gemm(m, n, k, gz.DT_BF16, gz.DT_F32, layout_b=gz.COL_MAJOR, config=config)
    d = torch.zeros(m, n, device="cuda")
    g.plan.run_ex(a, b, None, d, 1.0, 0.0, activation=ACTS[act])
    torch.cuda.synchronize()
    assert g.plan.device_status()[0] == api.GZ_OK
    want = np.zeros((m, n), dtype=bool)
    want[r], want[:, c] = True, True
    assert np.array_equal(torch.isnan(d).cpu().numpy(), want)
    if act == "relu":
        exact = np.maximum(a.cpu().double().numpy() @ b.cpu().double().numpy().T, 0)
        assert np.array_equal(d.cpu().double().numpy()[~want], exact[~want])
